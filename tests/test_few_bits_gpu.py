"""Models whose keys and values are kept in 4 bits and whose products run in 8-bit integers, as a user has them: through the engine, eager and captured, in portions and single tokens.

The oracle computes in 64 bits.  What the engine rounded to few bits (kept keys and values, rows in 8 bits) is checked against the oracle's own value, half a step off at most, and then
takes its place: a value that lies between two codes may go either way, and what follows is judged by what was kept."""

from __future__ import annotations

import math

import pytest
import torch

import plain_llama as pl
from tiny import BF16_ULP, random_tokens

pytestmark = pytest.mark.gpu

BASE = dict(architectures=["LlamaForCausalLM"], model_type="llama", num_hidden_layers=2, rms_norm_eps=1e-5, rope_theta=10000.0, max_position_embeddings=4096, tie_word_embeddings=False)
# head sizes 64 and 128 have attention on the matrix cores, 32 has not; groups of 3, 20 and 4 query heads
CONFIGS = {
    "head64": dict(BASE, vocab_size=500, hidden_size=192, intermediate_size=304, num_attention_heads=6, num_key_value_heads=2, head_dim=64),
    "head128": dict(BASE, vocab_size=311, hidden_size=256, intermediate_size=520, num_attention_heads=20, num_key_value_heads=1, head_dim=128),
    "head32": dict(BASE, vocab_size=400, hidden_size=128, intermediate_size=272, num_attention_heads=4, num_key_value_heads=1, head_dim=32),
}
PAGE = {"head64": 16, "head128": 8, "head32": 32}
# logits in terms of their row's largest, as for models in plain precision; what is rounded to few bits in terms of its row's largest: the errors that gather in the stream before it
LOGITS = {torch.float32: 1e-4, torch.bfloat16: 8 * BF16_ULP}
SLACK = {torch.float32: 1e-4, torch.bfloat16: 2.0**-5}


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    from nanospec_amd.config import LlamaConfig
    from nanospec_amd.weights import write_model_folder

    base = tmp_path_factory.mktemp("few_bits")
    return {name: write_model_folder(base / name, LlamaConfig.from_hf(cfg), 3, torch.float32) for name, cfg in CONFIGS.items()}


_MODELS: dict = {}


def model_of(folders, name, dtype, products="model", layouts="auto"):
    from nanospec_amd import load_model

    key = (name, dtype, products, layouts)
    if key not in _MODELS:
        _MODELS[key] = load_model(folders[name], dtype=dtype, products=products, layouts=layouts)
    return _MODELS[key]


def weight_in_8_bits(w):
    """float32 [N, K] -> what its codes stand for, float64."""
    most = w.abs().amax(1, keepdim=True)
    return torch.round(w * (127.0 / most)).clamp(-127, 127).double() * (most / 127).double()


class Oracle:
    def __init__(self, folder, dtype, products):
        self.cfg, w = pl.read_config(folder), pl.read_weights(folder, dtype)
        self.dtype, self.products = dtype, products
        of_layers = lambda name: products == "int8" and ".layers." in name and name.endswith("proj.weight")
        self.w = {k: weight_in_8_bits(v.float()) if of_layers(k) else v.double() for k, v in w.items()}

    def rows(self, x, given, at):
        """x as the product reads it: the engine's codes, each within half a step."""
        if given is None:
            return x
        codes, scales = given[at]
        most = x.abs().amax(1, keepdim=True)
        assert ((scales[:, None] * 127 - most).abs() <= SLACK[self.dtype] * most).all()
        off = (x - codes * scales[:, None]).abs() / most
        assert float(off.max()) <= 0.5 / 127 + 2 * SLACK[self.dtype], f"rows {at}: {float(off.max()) * 127} steps off"
        return codes * scales[:, None]

    def kept(self, x, given):
        """x [tokens, heads, dim] as the attention reads it: what the pages hold, within half a step."""
        if given is None:
            return x
        low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
        step = (high - low + 2.0**-7 * low.abs()) / 15 * (1 + 2.0**-7)
        bound = step / 2 + SLACK[self.dtype] * x.abs().amax(-1, keepdim=True)
        assert ((given - x).abs() <= bound).all(), "a kept key or value is more than half a step off"
        assert float((given - x).abs().max()) > 0  # (it is in 4 bits indeed)
        return given

    def __call__(self, tokens, kept=None, rows=None):
        """Logits [T, vocab] of a sequence.  ``kept``: per layer (keys, values) [T, kv_heads, dim]; ``rows``: per layer four (codes [T, K], scales [T])."""
        c, w, T = self.cfg, self.w, len(tokens)
        norm = lambda x, weight: weight * x * torch.rsqrt((x * x).mean(-1, keepdim=True) + c["eps"])
        x = w["model.embed_tokens.weight"][torch.tensor(tokens)]
        cos, sin = pl.rotation_tables(torch.arange(T), pl.inverse_frequencies(c["head_dim"], c["theta"], c["scaling"]))
        cos, sin, half = cos.double()[:, None], sin.double()[:, None], c["head_dim"] // 2
        rotate = lambda y: y * cos + torch.cat((-y[..., half:], y[..., :half]), -1) * sin
        hidden = torch.arange(T)[None] > torch.arange(T)[:, None]
        for i in range(c["layers"]):
            p = f"model.layers.{i}."
            given = None if rows is None else rows[i]
            h = self.rows(norm(x, w[p + "input_layernorm.weight"]), given, 0)
            q, k, v = ((h @ w[p + f"self_attn.{n}_proj.weight"].T).view(T, -1, c["head_dim"]) for n in "qkv")
            q, k = rotate(q), rotate(k)
            if kept is not None:
                k, v = self.kept(k, kept[i][0]), self.kept(v, kept[i][1])
            group = c["heads"] // c["kv_heads"]
            k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
            s = torch.einsum("qhd,khd->hqk", q, k) / math.sqrt(c["head_dim"])
            a = torch.einsum("hqk,khd->qhd", torch.softmax(s.masked_fill(hidden, -math.inf), -1), v).reshape(T, -1)
            x = x + self.rows(a, given, 1) @ w[p + "self_attn.o_proj.weight"].T
            h = self.rows(norm(x, w[p + "post_attention_layernorm.weight"]), given, 2)
            g, u = h @ w[p + "mlp.gate_proj.weight"].T, h @ w[p + "mlp.up_proj.weight"].T
            x = x + self.rows(g * torch.sigmoid(g) * u, given, 3) @ w[p + "mlp.down_proj.weight"].T
        return norm(x, w["model.norm.weight"]) @ w["lm_head.weight"].T


def kept_of(runner, storage, req_id, T):
    """What the cache keeps of a live request's first T tokens: per layer (keys, values), float64 on the CPU."""
    rc = runner.manager.get(req_id)
    runner.synchronize()
    out = []
    for entry, view in enumerate(storage.views):
        table = torch.tensor([rc.tables[view.group]], dtype=torch.int32, device="cuda")
        k, v = storage.kept(entry, torch.arange(T, dtype=torch.int32, device="cuda"), torch.zeros(T, dtype=torch.int32, device="cuda"), table)
        out.append((k.double().cpu(), v.double().cpu()))
    return out


def assert_logits(ours, ref, dtype, what):
    err = ((ours.double() - ref).abs().amax(-1) / ref.abs().amax(-1)).max()
    assert float(err) <= LOGITS[dtype], f"{what}: logits off by {float(err):.2e} of the row's largest"


# steps of a trace: request -> tokens it brings.  Whole prompts, a portion beside single tokens, single tokens alone, portions that end inside pages.
TRACE = [{"a": 70, "b": 5, "c": 1}, {"b": 41, "a": 1}, {"a": 1, "b": 1, "c": 1}, {"c": 33}, {"a": 1, "b": 1}, {"a": 1, "c": 2, "b": 1}]


def run_trace(model, name, kv_format, use_graphs, after_step=None, rounds=1):
    """-> tokens of each request, the logits of its tokens by position, the replayer."""
    from nanospec_amd.engine.replay import Replayer

    rep = Replayer(model, 1024, PAGE[name], use_graphs, kv_format=kv_format)
    vocab = CONFIGS[name]["vocab_size"]
    tokens, logits = {r: [] for r in "abc"}, {r: {} for r in "abc"}
    for n, step in enumerate(TRACE * rounds):
        entries = []
        for r, m in step.items():
            new = random_tokens(m, vocab, 100 * n + ord(r))
            entries.append({"id": r, "tokens": new, "want": [m - 1]})
            tokens[r] += new
        out = rep.step(entries, [])
        for row, r in zip(out, step):
            logits[r][len(tokens[r]) - 1] = row
        if after_step:
            after_step(step, tokens)
    return tokens, logits, rep


@pytest.mark.parametrize("use_graphs", [False, True], ids=["eager", "captured"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("name", CONFIGS)
def test_keys_and_values_in_4_bits(folders, name, dtype, use_graphs):
    """Prompts, portions and single tokens over one cache: what is kept is half a step off at most, and the logits are those of what is kept."""
    model = model_of(folders, name, dtype)
    tokens, logits, rep = run_trace(model, name, "int4", use_graphs, rounds=3)
    oracle = Oracle(folders[name], dtype, "model")
    for r in "abc":
        ref = oracle(tokens[r], kept=kept_of(rep.runner, rep.storage, r, len(tokens[r])))
        at = sorted(logits[r])
        assert_logits(torch.stack([logits[r][i] for i in at]), ref[at], dtype, f"request {r}")


def recorded(monkeypatch):
    """Every row in 8 bits that a step makes, in order."""
    from nanospec_amd.kernels import ops

    made = []

    def keep(fn):
        def wrapped(*args, **kw):
            rows = fn(*args, **kw)
            made.append((rows.codes().double().cpu(), rows.scales.double().cpu()))
            return rows
        return wrapped

    for name in ("rmsnorm_int8", "int8_rows", "silu_mul_int8"):
        monkeypatch.setattr(ops, name, keep(getattr(ops, name)))
    return made


@pytest.mark.parametrize("kv_format", ["int4", "model"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("name", CONFIGS)
def test_products_in_8_bits(folders, name, dtype, kv_format, monkeypatch):
    """With and without the 4-bit cache: every row that a product reads is half a step off at most, and the logits are those of the rows that were read."""
    model = model_of(folders, name, dtype, "int8")
    layers = CONFIGS[name]["num_hidden_layers"]
    made = recorded(monkeypatch)
    rows = {r: [[[] for _ in range(4)] for _ in range(layers)] for r in "abc"}

    def sort(step, _tokens):
        assert len(made) == 4 * layers
        for i, (codes, scales) in enumerate(made):
            at = 0
            for r, m in step.items():
                rows[r][i // 4][i % 4].append((codes[at : at + m], scales[at : at + m]))
                at += m
        made.clear()

    tokens, logits, rep = run_trace(model, name, kv_format, False, after_step=sort)
    oracle = Oracle(folders[name], dtype, "int8")
    for r in "abc":
        whole = [[tuple(torch.cat(t) for t in zip(*pieces)) for pieces in layer] for layer in rows[r]]
        kept = kept_of(rep.runner, rep.storage, r, len(tokens[r])) if kv_format == "int4" else None
        ref = oracle(tokens[r], kept=kept, rows=whole)
        at = sorted(logits[r])
        assert_logits(torch.stack([logits[r][i] for i in at]), ref[at], dtype, f"request {r}")


@pytest.mark.parametrize("name", CONFIGS)
def test_captured_steps_of_few_bits(folders, name):
    """Graphs of steps with both, replayed with eager work between: the logits of the eager run.  A value between two codes may go the other way where attention's ranges are cut otherwise:
    of a row of K codes some four
    are moved by a step, 1/127 of the row's largest, which is at most five times its typical value: 2 * 5 / (127 sqrt(K)) of the product, 0.7% at K = 128; over 8 products that is 2%, and with
    as much again from the cache, as squares add, 2.8% of the largest logit."""
    model = model_of(folders, name, torch.float32, "int8")
    eager = run_trace(model, name, "int4", False, rounds=3)
    captured = run_trace(model, name, "int4", True, after_step=lambda step, tokens: torch.randn(1000, device="cuda").sum().item(), rounds=3)
    assert eager[0] == captured[0]
    for r in "abc":
        for i, row in eager[1][r].items():
            assert float((captured[1][r][i] - row).abs().max() / row.abs().max()) <= 0.03


@pytest.mark.parametrize("products", ["model", "int8"])
def test_through_the_engine(folders, products):
    """Continuous batching, portions, lookahead and captured steps, and a pool that is too small: every request gets its tokens and no page is lost; greedy tokens are the arg-max of the
    logits that their step recorded."""
    from nanospec_amd import Engine, EngineConfig, SamplingParams

    name = "head64"
    model = model_of(folders, name, torch.bfloat16, products)
    prompts = [random_tokens(n, 500, n) for n in (3, 40, 17, 90, 1, 64)]
    for options in (dict(num_blocks=128), dict(num_blocks=128, cuda_graphs=False, prefill_chunk=23, max_step_tokens=48),
                    dict(num_blocks=14, on_exhaustion="preempt", prefill_chunk=32)):
        eng = Engine(model, EngineConfig(block_size=16, kv_format="int4", **options))
        outs = eng.generate(prompts, SamplingParams(max_tokens=20))
        assert all(len(o) == 20 and all(0 <= t < 500 for t in o) for o in outs)
        eng.cache.check()
        assert eng.cache.num_free() == eng.usable_blocks
    eng = Engine(model, EngineConfig(block_size=16, kv_format="int4", num_blocks=128, record_logits=True))
    reqs = [eng.add(p, SamplingParams(max_tokens=8)) for p in prompts]
    while eng.sched.has_work:
        eng.step()
    for r in reqs:
        assert [int(t.argmax()) for t in r.step_logits] == r.out_tokens


def test_generate_and_command_line(folders):
    import json
    import subprocess
    import sys
    from pathlib import Path

    from nanospec_amd import SamplingParams, generate

    folder, prompt = str(folders["head128"]), random_tokens(20, 311, 5)
    out = generate(folder, [prompt], SamplingParams(max_tokens=6), products="int8", kv_format="int4")
    proc = subprocess.run([sys.executable, "-m", "nanospec_amd", "--model", folder, "--max-tokens", "6", "--products", "int8", "--kv-format", "int4", "--prompt-ids",
                           ",".join(map(str, prompt))], capture_output=True, text=True, cwd=Path(__file__).resolve().parent.parent, timeout=600)
    assert proc.returncode == 0, proc.stderr[-2000:]
    assert json.loads(proc.stdout)["output_ids"] == out[0] and len(out[0]) == 6
    with pytest.raises(ValueError, match="chosen as a model is loaded"):
        generate(model_of(folders, "head128", torch.bfloat16), [prompt], products="int8")


@pytest.mark.parametrize("layouts", ["both", "tiled"])
def test_a_model_serves_both_formats(folders, layouts):
    """One model, an engine in its own precision before and after one in 4 bits: its results are the same bits."""
    model = model_of(folders, "head64", torch.bfloat16, layouts=layouts)
    before = run_trace(model, "head64", "model", True)
    few = run_trace(model, "head64", "int4", True)
    after = run_trace(model, "head64", "model", True)
    differ = 0
    for r in "abc":
        for i, row in before[1][r].items():
            assert torch.equal(row, after[1][r][i])
            differ += not torch.equal(row, few[1][r][i])
    assert differ


def test_what_a_cache_in_4_bits_takes(folders):
    model = model_of(folders, "head64", torch.bfloat16)
    from nanospec_amd.cache.storage import CacheStorage

    few, full = (CacheStorage(model, [8], 16, 4, torch.bfloat16, "cuda", f) for f in ("int4", "model"))
    # 2 layers of 2 heads of keys and values of 64 channels: 4 bits each and 4 bytes a key or value
    assert few.bytes_per_token() == 2 * 2 * 2 * (32 + 4) and full.bytes_per_token() == 2 * 2 * 2 * 128
    assert few.int4[0].numel() == 8 * 16 * few.bytes_per_token()
    t = torch.arange(40, dtype=torch.int32, device="cuda")
    table = torch.tensor([[3, 1, 2]], dtype=torch.int32, device="cuda")
    for storage in (few, full):
        k, v = storage.kept(1, t, torch.zeros_like(t), table)
        assert k.shape == v.shape == (40, 2, 64) and not k.any() and not v.any()  # pages of zeros stand for zeros


def _wide(tmp_path_factory):
    """A folder whose q/k/v matrices are large enough to be counted: 4 layers of 1,536 x 1,024, 3 MiB each in bfloat16."""
    from nanospec_amd.config import LlamaConfig
    from nanospec_amd.weights import write_model_folder

    cfg = dict(BASE, num_hidden_layers=4, vocab_size=300, hidden_size=1024, intermediate_size=512, num_attention_heads=16, num_key_value_heads=4, head_dim=64)
    return write_model_folder(tmp_path_factory.mktemp("wide"), LlamaConfig.from_hf(cfg), 3, torch.float32)


def _allocated():
    import gc

    gc.collect()
    torch.cuda.synchronize()
    return torch.cuda.memory_allocated()


def test_a_cache_in_4_bits_leaves_a_model_as_it_was(tmp_path_factory):
    """The copies of the q/k/v matrices that layers run over such a cache belong to it: two caches share them, and the last one takes them along."""
    from nanospec_amd import load_model
    from nanospec_amd.cache.storage import CacheStorage

    model = load_model(_wide(tmp_path_factory), layouts="both")
    before, copies = _allocated(), 4 * 1536 * 1024 * 2
    make = lambda: CacheStorage(model, [8], 16, 4, torch.bfloat16, "cuda", "int4")
    one = make()
    pages = sum(t.numel() for t in one.int4)
    first = _allocated()
    assert len(one.products) == 4 and copies <= first - before - pages < 1.5 * copies
    two = make()
    assert _allocated() - first < pages + copies / 8 and all(two.products[k] is v for k, v in one.products.items())
    del one
    assert all(p is not None for p in two.products.values()) and _allocated() - before >= copies
    del two
    assert _allocated() - before < copies / 8


@pytest.mark.parametrize("fails", ["pages", "copies"])
def test_a_cache_in_4_bits_where_memory_is_short(tmp_path_factory, monkeypatch, fails, capsys):
    """No room beside two copies of the q/k/v matrices: the layers keep one, and serve either cache with it."""
    from nanospec_amd import load_model
    from nanospec_amd.cache.storage import CacheStorage
    from nanospec_amd.engine.replay import Replayer
    from nanospec_amd.parts.attention import Attention

    folder = _wide(tmp_path_factory)
    model, other = load_model(folder, layouts="both"), load_model(folder, layouts="both")
    before = _allocated()
    owner, name = (CacheStorage, "_allocate") if fails == "pages" else (Attention, "serve_int4_cache")
    plain, calls = getattr(owner, name), []

    def short(self, *args, **kw):
        calls.append(self)
        if len(calls) == (1 if fails == "pages" else 3):
            raise torch.OutOfMemoryError("no room")
        return plain(self, *args, **kw)

    monkeypatch.setattr(owner, name, short)
    rep = Replayer(model, 512, 16, True, kv_format="int4")
    monkeypatch.undo()
    assert not rep.storage.products and all(layer.mixer.wqkv_rope is None and layer.mixer.wqkv.tiled is not None for layer in model.layers)
    assert "in one order" in capsys.readouterr().err
    steps = [[{"id": "a", "tokens": random_tokens(n, 300, n + i), "want": [n - 1]}] for i, n in enumerate((40, 1, 1, 200, 1))]
    for kv_format, made in (("int4", rep), ("model", Replayer(model, 512, 16, True))):
        whole = Replayer(other, 512, 16, True, kv_format=kv_format)
        assert kv_format == "model" or len(whole.storage.products) == 4
        for step in steps:
            a, b = made.step(step, []), whole.step(step, [])
            # other kernels' roundings of q, k and v; a value between two codes may go the other way (0.03, as for captured steps; in bfloat16 8 units of the row's largest besides)
            assert float((a - b).abs().max() / b.abs().max()) <= 0.03 + LOGITS[torch.bfloat16]
    del rep, whole, made, a, b
    assert not other.stream_one_order({}) and all(layer.mixer.wqkv_rope is not None for layer in other.layers)  # (it has run)


def test_a_model_with_one_copy_has_none_to_give(tmp_path_factory, monkeypatch, capsys):
    """In the tiled layout layers run their own product over either cache: nothing is made for one in 4 bits, and where its pages do not fit nothing changes."""
    from nanospec_amd import load_model
    from nanospec_amd.cache.storage import CacheStorage

    model = load_model(_wide(tmp_path_factory), layouts="tiled")
    capsys.readouterr()
    plain, calls = CacheStorage._allocate, []

    def short(self, *args, **kw):
        calls.append(self)
        if len(calls) == 1:
            raise torch.OutOfMemoryError("no room")
        return plain(self, *args, **kw)

    monkeypatch.setattr(CacheStorage, "_allocate", short)
    storage = CacheStorage(model, [8], 16, 4, torch.bfloat16, "cuda", "int4")
    assert len(calls) == 2 and not storage.products and storage.views[0].products is storage.products
    assert all(layer.mixer.wqkv_rope is not None for layer in model.layers) and not capsys.readouterr().err

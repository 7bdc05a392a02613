"""Operands in 8 bits on the CPU: the layout, and what is refused."""

from __future__ import annotations

import pytest
import torch

from nanospec_amd.kernels import ops


@pytest.mark.parametrize("n,k", [(1, 1), (16, 512), (37, 700), (48, 1024)])
def test_layout(n, k):
    codes = torch.randint(-127, 128, (n, k), dtype=torch.int8, generator=torch.Generator().manual_seed(n))
    w = ops.Int8Weight(codes, torch.arange(n, dtype=torch.float32))
    assert torch.equal(w.codes(), codes) and w.kp % 256 == 0 and w.kp >= max(512, k) and torch.equal(w.scales[:n], torch.arange(n, dtype=torch.float32))
    flat = w.data.reshape(-1)
    for row, col in ((0, 0), (n - 1, k - 1), (n // 2, k // 2), (n // 3, k // 3)):
        at = ((row // 16) * (w.kp // 64) + col // 64) * 1024 + (16 * (col % 64 // 16) + row % 16) * 16 + col % 16
        assert flat[at] == codes[row, col]
    assert int(w.data.abs().long().sum()) == int(codes.abs().long().sum())  # zeros everywhere else


@pytest.mark.parametrize("m,k", [(0, 64), (1, 1), (16, 700), (17, 512)])
def test_room_for_rows(m, k):
    for take in (None, lambda shape, dtype: torch.empty(shape, dtype=dtype)):
        rows = ops.Int8Rows._made(m, k, torch.device("cpu"), take)
        rows.whole.copy_(torch.arange(rows.whole.numel()) % 100)
        assert rows.data.shape == (-(-m // 16), ops.int8_padded_k(k) // 64, 4, 16, 16) and rows.scales.shape == (m,) and rows.codes().shape == (m, k)
        assert rows.data.numel() + 4 * m == rows.whole.numel() and rows.scales.dtype == torch.float32
        if m:
            assert rows.scales.data_ptr() == rows.data.data_ptr() + rows.data.numel()


def test_from_float_keeps_rows_apart():
    w = torch.tensor([[1.0, -2.0, 0.5], [0.0, 0.0, 0.0], [float("inf"), 1.0, 0.0], [float("nan"), 1.0, 0.0], [2.0**-110, 0.0, 0.0]])
    made = ops.Int8Weight.from_float(w)
    assert made.codes()[0].tolist() == [64, -127, 32] and not bool(made.codes()[1:].any())
    assert float(made.scales[0]) == 2 / 127 or abs(float(made.scales[0]) - 2 / 127) < 1e-9
    assert made.scales[1] == 0 and made.scales[4] == 0 and bool(torch.isnan(made.scales[2:4]).all())


@pytest.mark.parametrize("codes,scales", [(torch.zeros(4, 8), torch.zeros(4)), (torch.zeros(4, 8, dtype=torch.int8), torch.zeros(3)), (torch.zeros(4, 8, dtype=torch.int8), torch.zeros(4).double()),
                                          (torch.zeros(4, dtype=torch.int8), torch.zeros(4)), (torch.zeros(1, 32769, dtype=torch.int8), torch.zeros(1)), (torch.zeros(0, 8, dtype=torch.int8), torch.zeros(0))])
def test_weights_that_are_refused(codes, scales):
    with pytest.raises(ops.KernelRefused):
        ops.Int8Weight(codes, scales)


def test_rows_that_are_refused(monkeypatch):
    x = torch.zeros(3, 64)
    for call in (lambda: ops.int8_rows(x), lambda: ops.silu_mul_int8(x), lambda: ops.rmsnorm_int8(torch.ones(64), 1e-5, x=x)):
        with pytest.raises(ops.KernelRefused, match="GPU"):
            call()
    monkeypatch.setattr(ops, "_gpu", lambda *tensors: None)
    one = torch.ones(64)
    for call in (lambda: ops.int8_rows(x[0]), lambda: ops.int8_rows(x.t()), lambda: ops.int8_rows(torch.zeros(1, 32769)), lambda: ops.int8_rows(x.half()), lambda: ops.int8_rows(x[:, :0]),
                 lambda: ops.int8_rows(x[:1].expand(3, 64)), lambda: ops.silu_mul_int8(torch.zeros(3, 63)), lambda: ops.rmsnorm_int8(one, 1e-5),
                 lambda: ops.rmsnorm_int8(one, 1e-5, x=x, resid=torch.zeros(2, 64)), lambda: ops.rmsnorm_int8(one, 1e-5, x=x, resid=x.bfloat16()), lambda: ops.rmsnorm_int8(one[:32], 1e-5, x=x),
                 lambda: ops.rmsnorm_int8(one, 1e-5, x=x, resid_out=torch.zeros(3, 128)[:, :64])):
        with pytest.raises(ops.KernelRefused):
            call()


def test_products_that_are_refused(monkeypatch):
    monkeypatch.setattr(ops, "_gpu", lambda *tensors: None)
    w = ops.Int8Weight(torch.zeros((48, 600), dtype=torch.int8), torch.zeros(48))
    rows = ops.Int8Rows.from_codes(torch.zeros((3, 600), dtype=torch.int8), torch.zeros(3))
    for call in (lambda: ops.linear_int8(torch.zeros(3, 600), w), lambda: ops.linear_int8(rows, torch.zeros(48, 600)), lambda: ops.linear_int8(rows, w, out=torch.zeros(3, 47)),
                 lambda: ops.linear_int8(rows, w, out=torch.zeros(48, 3).t()), lambda: ops.linear_int8(rows, w, dtype=torch.float16),
                 lambda: ops.linear_int8(ops.Int8Rows(rows.data, rows.scales, 601), w), lambda: ops.linear_int8(ops.Int8Rows(rows.data, torch.zeros(17), 600), w), lambda: ops.linear_int8(ops.Int8Rows(rows.data, torch.zeros(6)[::2], 600), w),
                 lambda: ops.linear_int8(ops.Int8Rows(rows.data[:, :8], rows.scales, 600), w), lambda: ops.linear_int8(ops.Int8Rows(rows.data.float(), rows.scales, 600), w),
                 lambda: ops.Int8Rows.from_codes(torch.zeros(3, 600), torch.zeros(3)), lambda: ops.Int8Rows.from_codes(torch.zeros((3, 600), dtype=torch.int8), torch.zeros(2))):
        with pytest.raises(ops.KernelRefused):
            call()


def test_plan():
    """Few rows, or little to read, go by row blocks; ranges of K are as long as a tile takes at least; pieces are whole tiles' columns and make up the product; a plan stands for every size."""
    few = lambda *sizes: ops.int8_plan(*sizes, 256)[0][1] < 0
    assert few(1, 28672, 4096) and few(16, 28672, 4096) and few(32, 4096, 4096) and not few(48, 28672, 4096) and not few(2048, 4096, 4096)
    assert len(ops.int8_plan(2048, 28672, 4096, 256)) == 2
    for m in (17, 100, 999, 4096, 70000):
        for n in (1, 1000, 4096, 10007, 28672, 128256):
            for k in (1, 513, 4096, 32768):
                pieces = ops.int8_plan(m, n, k, 256)
                assert sum(c for c, _, _ in pieces) == n and len(pieces) <= 2
                for i, (columns, form, ranges) in enumerate(pieces):
                    if form < 0:
                        assert -form in (1, 2, 4) and ranges == 1 and -(-m // (-16 * form)) <= 65535
                        continue
                    assert form < len(ops.INT8_TILES) and ops.int8_padded_k(k) >= ranges * ops.INT8_K_MIN
                    assert i == len(pieces) - 1 or columns % ops.INT8_TILES[form][1] == 0
                    tiles = -(-m // ops.INT8_TILES[form][0]) * -(-columns // ops.INT8_TILES[form][1])
                    assert tiles * ranges <= 1 << 22


def test_models_refuse_products_that_are_not_built():
    """Before anything is read or moved."""
    from types import SimpleNamespace

    from nanospec_amd.config import LlamaConfig
    from nanospec_amd.parts import DecoderModel
    from tiny import TINY

    net = DecoderModel(LlamaConfig.from_hf(TINY["A"]["cfg"]).model_spec())
    with pytest.raises(ValueError, match="products="):
        net.load(None, torch.float32, "cpu", products="int4")
    from nanospec_amd.config import VuzelixConfig
    from test_vuzelix_config import CFG

    with pytest.raises(ValueError, match="not built for StreamBlock"):
        DecoderModel(VuzelixConfig.from_hf(CFG).model_spec()).load(None, torch.float32, "cpu", products="int8")
    net.layers[1].ffn = SimpleNamespace()
    with pytest.raises(ValueError, match="not built for SimpleNamespace"):
        net.load(None, torch.float32, "cpu", products="int8")


def test_plans_of_more_rows_than_are_joined():
    for m in (65535, 65536, 200_000):
        for n, k in ((17, 32768), (64, 8192), (4096, 4096)):
            plan = ops.int8_plan(m, n, k, 256)
            assert all(ranges == 1 or m <= ops.INT8_JOIN_ROWS for _, _, ranges in plan)


def test_models_refuse_layers_and_sizes_before_anything_is_read():
    """Layers of the right kinds with options that have no products in 8-bit integers, and inner sizes that those do not sum over: by the layer's number, with nothing to read from."""
    from nanospec_amd.config import LlamaConfig
    from nanospec_amd.parts import DecoderModel
    from tiny import TINY

    cfg = TINY["A"]["cfg"]
    fresh = lambda **change: DecoderModel(LlamaConfig.from_hf({**cfg, **change}).model_spec())
    for change, what in ((dict(intermediate_size=32784), "layer 0: a feed-forward.*32768 values, not 32784"), (dict(hidden_size=32832), "layer 0: an attention layer.*not 32832"),
                         (dict(num_attention_heads=2050, num_key_value_heads=2), "layer 0: an attention layer.*not 32800")):
        with pytest.raises(ValueError, match=what):
            fresh(**change).load(None, torch.float32, "cpu", products="int8")
    net = fresh()
    net.layers[1].ffn.biased = True
    with pytest.raises(ValueError, match="layer 1: a feed-forward with biases"):
        net.load(None, torch.float32, "cpu", products="int8")
    import dataclasses

    net = fresh()
    net.layers[1].mixer.spec = dataclasses.replace(net.layers[1].mixer.spec, sink=True)
    assert net.layers[1].mixer.spec.general
    with pytest.raises(ValueError, match="layer 1: an attention layer with options"):
        net.load(None, torch.float32, "cpu", products="int8")
    # what these sizes are refused for is the products alone
    with pytest.raises(AttributeError):
        fresh(intermediate_size=32784).load(None, torch.float32, "cpu")

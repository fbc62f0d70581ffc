"""MXFP4 layers, checkpoints and operators on the CPU: what they hold and refuse."""

import json

import pytest
import torch

import mlxturbo_amd as mq
from mlxturbo_amd import _lib, checkpoint, nn, ops, rebit

KW = dict(mode="mxfp4")


@pytest.fixture
def on_cpu(monkeypatch):
    """Argument checks with CPU tensors; the library is not called."""
    monkeypatch.setattr(ops, "_require_gpu", lambda *ts: torch.device("cpu"))

    class NoLib:
        def __getattr__(self, name):
            raise AssertionError(f"{name} called")
    monkeypatch.setattr(_lib, "lib", NoLib)


def _w(N=48, K=256, E=None):
    lead = (E, N) if E else (N,)
    return (torch.zeros(*lead, K // 8, dtype=torch.int32),
            torch.zeros(*lead, K // 32, dtype=torch.uint8))


@pytest.mark.parametrize("key", ["torch_dtype", "dtype"])
def test_checkpoint_float_type(tmp_path, key):
    from safetensors.torch import save_file
    w, s = _w()
    save_file({"a.weight": w.view(torch.uint32), "a.scales": s,
               "e.weight": _w(E=2)[0].view(torch.uint32), "e.scales": _w(E=2)[1]},
              str(tmp_path / "model.safetensors"))
    for named, want in (("float16", torch.float16), ("other", torch.bfloat16),
                        (None, torch.bfloat16)):
        cfg = {"quantization": {"group_size": 32, "bits": 4, "mode": "mxfp4"}, key: named}
        (tmp_path / "config.json").write_text(json.dumps(cfg))
        layers = checkpoint.quantized_layers(str(tmp_path), device="cpu")
        assert layers["a"]._like.dtype == want and layers["e"].mode == "mxfp4"


def test_affine_layers_have_their_scales_type():
    w, s = torch.zeros(8, 32, dtype=torch.int32), torch.zeros(8, 4, dtype=torch.float16)
    assert nn.QuantizedLinear(w, s, s, dtype=torch.float16).mode == "affine"
    with pytest.raises(ValueError, match="scales' dtype"):
        nn.QuantizedLinear(w, s, s, dtype=torch.bfloat16)


def test_requantize_takes_the_modes_own_group_size(monkeypatch):
    seen = []
    monkeypatch.setattr(nn.QuantizedLinear, "from_linear",
                        classmethod(lambda cls, w, bias=None, **kw: seen.append(kw)))
    lin = torch.nn.Linear(96, 8, bias=False)
    rebit.requantize(lin, 4, mode="mxfp4")               # 96 is groups of 32 alone
    rebit.requantize(torch.nn.Linear(128, 8), 8)
    rebit.requantize(lin, 8, 32)
    assert seen == [dict(group_size=32, bits=4, mode="mxfp4"),
                    dict(group_size=64, bits=8, mode="affine"),
                    dict(group_size=32, bits=8, mode="affine")]
    with pytest.raises(ValueError, match="multiple of group_size=64"):
        rebit.requantize(lin, 8)
    for bad in (dict(bits=4, group_size=64), dict(bits=8)):
        with pytest.raises(ValueError, match="groups of 32"):
            rebit.requantize(lin, mode="mxfp4", **bad)


@pytest.mark.parametrize("E,N", [(3, 1), (2, 48), (1, 48)])
def test_gate_and_up_banks_of_other_shapes_are_refused(on_cpu, E, N):
    gate, up = (*_w(E=3), None), (*_w(E=E, N=N), None)
    x = torch.zeros(4, 1, 1, 256, dtype=torch.bfloat16)
    idx = torch.zeros(4, 2, dtype=torch.int32)
    wts = torch.zeros(4, 2)
    with pytest.raises(ValueError, match="banks differ in shape"):
        mq.gather_glu(x, *gate, *up, rhs_indices=idx, **KW)
    with pytest.raises(ValueError, match="banks differ in shape"):
        ops.gather_swiglu(x, gate, up, idx, None, **KW)
    with pytest.raises(ValueError, match="banks differ in shape"):
        ops.moe_layer(x.reshape(4, 256), idx, wts, gate, up, (*_w(E=3, N=256, K=64), None), **KW)


@pytest.mark.parametrize("E", [None, 3])
def test_layers_hold_scale_bytes(E):
    """float8_e8m0fnu scales are the same bytes as uint8 ones, through the module's
    conversions and state dicts of either type."""
    cls = nn.QuantizedSwitchLinear if E else nn.QuantizedLinear
    w, s = _w(E=E)
    s = torch.randint(0, 256, s.shape, dtype=torch.uint8)
    e8 = s.view(torch.float8_e8m0fnu)
    lin = torch.nn.ModuleDict({"a": cls(w, e8, None, **KW)})
    assert torch.equal(lin["a"].scales, s)
    assert torch.equal(lin.half()["a"].scales, s)
    for assign in (False, True):
        for given in (s, e8):
            new = torch.nn.ModuleDict({"a": cls(w, torch.zeros_like(s), None, **KW)})
            state = {"a.weight": w, "a.scales": given}
            new.load_state_dict(state, assign=assign)
            assert torch.equal(new["a"].scales, s) and state["a.scales"] is given
    aff = nn.QuantizedLinear(torch.zeros(8, 32, dtype=torch.int32), *[torch.zeros(8, 4)] * 2)
    aff.load_state_dict({"weight": aff.weight, "scales": torch.ones(8, 4, dtype=torch.float16),
                         "biases": torch.ones(8, 4)})
    assert aff.scales.dtype == torch.float32 and bool((aff.scales == 1).all())


def test_checkpoint_width_from_the_shapes_is_affine(tmp_path):
    """A module without an entry and of another width, in an MXFP4 checkpoint."""
    from safetensors.torch import save_file
    w, s = _w()
    b16 = torch.zeros(48, 8, dtype=torch.bfloat16)
    save_file({"a.weight": w.view(torch.uint32), "a.scales": s,
               "h.weight": torch.zeros(48, 64, dtype=torch.int32).view(torch.uint32),
               "h.scales": b16, "h.biases": b16.clone()}, str(tmp_path / "model.safetensors"))
    (tmp_path / "config.json").write_text(json.dumps({"quantization": {"mode": "mxfp4"}}))
    layers = checkpoint.quantized_layers(str(tmp_path), device="cpu")
    assert layers["a"].mode == "mxfp4"
    h = layers["h"]
    assert (h.mode, h.bits, h.group_size, h.input_dims) == ("affine", 8, 32, 256)


def test_checkpoint_bias_has_the_float_type(tmp_path):
    from safetensors.torch import save_file
    w, s = _w()
    save_file({"a.weight": w.view(torch.uint32), "a.scales": s,
               "a.bias": torch.zeros(48, dtype=torch.float16)},
              str(tmp_path / "model.safetensors"))
    cfg = {"quantization": {"mode": "mxfp4"}, "torch_dtype": "bfloat16"}
    (tmp_path / "config.json").write_text(json.dumps(cfg))
    layers = checkpoint.quantized_layers(str(tmp_path), device="cpu")
    assert layers["a"]._like.dtype == torch.float16


def test_a_float32_bias_does_not_set_the_float_type(tmp_path):
    from safetensors.torch import save_file
    w, s = _w()
    bias = torch.zeros(48)
    assert nn.QuantizedLinear(w, s, None, bias, **KW)._like.dtype == torch.bfloat16
    save_file({"a.weight": w.view(torch.uint32), "a.scales": s, "a.bias": bias},
              str(tmp_path / "model.safetensors"))
    cfg = {"quantization": {"mode": "mxfp4"}, "torch_dtype": "float16"}
    (tmp_path / "config.json").write_text(json.dumps(cfg))
    layers = checkpoint.quantized_layers(str(tmp_path), device="cpu")
    assert layers["a"]._like.dtype == torch.float16

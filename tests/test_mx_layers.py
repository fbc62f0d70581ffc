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

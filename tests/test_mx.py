"""MXFP4 on the CPU: the tests' own definition, the C ABI's argument checks, the
operators' refusals, and what the modules, checkpoints and rebit specs say."""

import json
import os

import pytest
import torch

import mlxturbo_amd as mq
from mlxturbo_amd import _lib, checkpoint, dispatch, mx, nn, ops, rebit
from mx_helpers import pack, quantize_ref, unpack, values_ref

FAKE = 256  # aligned, never dereferenced: validation fails before any HIP call


def test_definition_by_hand():
    v = torch.zeros(1, 64)
    v[0, :9] = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -7.9])
    v[0, 32:35] = torch.tensor([0.0, -0.0, 2.0 ** -126])
    code, e = quantize_ref(v)
    # floor(log2 7.9) - 2 = 0; ties go to even codes, 7.9 saturates
    assert e.tolist() == [[127, 0]]
    assert code[0, :9].tolist() == [7, 0, 2, 2, 4, 4, 6, 6, 15]
    # e = -126 - 2 clamps to -127: the value is 2 scales
    assert code[0, 32:35].tolist() == [0, 8, 4]
    assert torch.equal(unpack(pack(code)), code)
    got = values_ref(code, e)[0, :9]
    assert got.tolist() == [6.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, -6.0]
    code, e = quantize_ref(torch.tensor([float("inf")] + [1.0] * 31)[None])
    assert e.item() == 255 and not code.any() and values_ref(code, e).isnan().all()


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        from mlxturbo_amd import build
        build.build()
    return _lib.lib()


@pytest.mark.parametrize("kw,code,needle", [
    (dict(w=None), -1, "non-null"), (dict(s=None), -1, "non-null"),
    (dict(x=None), -1, "non-null"), (dict(out=None), -1, "non-null"),
    (dict(K=48), -1, "multiple"), (dict(K=0), -1, "sizes"), (dict(N=-1), -1, "sizes"),
    (dict(M=-1), -1, "M"), (dict(M=1 << 31), -1, "M"), (dict(N=1 << 31), -1, "int32"),
    (dict(dtype=2), -2, "float32"), (dict(dtype=7), -1, "dtype"),
    (dict(w=FAKE + 8), -1, "aligned"), (dict(s=FAKE + 4), -1, "aligned"),
    (dict(x=FAKE + 2), -1, "aligned"), (dict(out=FAKE + 1), -1, "aligned"),
])
@pytest.mark.parametrize("entry", ["matmul", "qqmm", "gather"])
def test_product_argument_validation(lib, entry, kw, code, needle):
    a = dict(x=FAKE, w=FAKE, s=FAKE, out=FAKE, M=1, N=16, K=64, dtype=0)
    a.update(kw)
    if entry == "gather":
        rc = lib.mq_mxfp4_gather_qmm(a["x"], a["w"], a["s"], None, FAKE, a["out"], 4, 4, a["M"],
                                     a["N"], a["K"], 2, a["dtype"], None, 0, None)
    else:
        f = lib.mq_mxfp4_matmul if entry == "matmul" else lib.mq_mxfp4_qqmm
        rc = f(a["x"], a["w"], a["s"], a["out"], a["M"], a["N"], a["K"], a["dtype"], None, 0, None)
    assert rc == code and needle in lib.mq_last_error().decode()


def test_format_argument_validation(lib):
    q, d = lib.mq_mxfp4_quantize, lib.mq_mxfp4_dequantize
    for f in (q, d):
        assert f(None, FAKE, FAKE, 4, 64, 0, None) == -1
        assert f(FAKE, FAKE, None, 4, 64, 0, None) == -1
        assert f(FAKE, FAKE, FAKE, 4, 40, 0, None) == -1
        assert f(FAKE, FAKE, FAKE, 4, 64, 3, None) == -1
        assert f(FAKE + 4, FAKE, FAKE, 4, 64, 0, None) == -1
        assert f(FAKE, FAKE, FAKE, 0, 64, 0, None) == 0


def test_gather_argument_validation(lib):
    def call(P=4, B=4, M=1, E=2, lhs=None, rhs=FAKE, ws=None, nb=0):
        return lib.mq_mxfp4_gather_qmm(FAKE, FAKE, FAKE, lhs, rhs, FAKE, P, B, M, 16, 64, E, 0, ws,
                                       nb, None)
    assert call(rhs=None) == -1
    assert call(P=4, B=3) == -1 and b"divide" in lib.mq_last_error()
    assert call(E=0) == -1 and call(M=17) == -2
    need = lib.mq_mxfp4_gather_qmm_workspace_size(2000, 1)
    assert need > 0 and call(P=2000, B=2000) == -1 and b"workspace" in lib.mq_last_error()
    assert call(P=2000, B=2000, ws=FAKE, nb=need - 1) == -1
    assert call(P=2000, B=2000, E=4096, ws=FAKE, nb=need) == -2
    assert lib.mq_mxfp4_gather_qmm_workspace_size(8, 1) == 0
    assert call(P=0) == 0 and call(M=0) == 0


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


def test_refusals(on_cpu):
    w, s = _w()
    x = torch.zeros(4, 256, dtype=torch.bfloat16)
    kw = dict(mode="mxfp4")
    with pytest.raises(NotImplementedError, match="biases"):
        mq.quantized_matmul(x, w, s, s, **kw)
    for bad in (dict(group_size=64), dict(bits=8)):
        with pytest.raises(ValueError, match="groups of 32"):
            mq.quantized_matmul(x, w, s, **kw, **bad)
        with pytest.raises(ValueError, match="groups of 32"):
            mq.quantize(x, **kw, **bad)
    with pytest.raises(ValueError, match="uint8"):
        mq.quantized_matmul(x, w, s.to(torch.bfloat16), **kw)
    with pytest.raises(ValueError, match="packed"):
        mq.quantized_matmul(x, w.float(), s, **kw)
    with pytest.raises(ValueError, match="scales shape"):
        mq.quantized_matmul(x, w, s[:, :4], **kw)
    with pytest.raises(ValueError, match="does not match"):
        mq.quantized_matmul(x[:, :128], w, s, **kw)
    with pytest.raises(ValueError, match="does not match"):
        mq.qqmm(x[:, :128], w, s)
    with pytest.raises(ValueError, match="take"):
        mq.quantized_matmul(x.double(), w, s, **kw)
    with pytest.raises(NotImplementedError, match="qqmm"):
        mq.qqmm(x, w, s, mode="affine")
    with pytest.raises(NotImplementedError, match="2-D"):
        mq.quantized_matmul(x, *_w(E=2), **kw)
    with pytest.raises(NotImplementedError):
        mq.quantized_matmul(x, w, s, mode="nvfp4")
    with pytest.raises(ValueError, match="multiple of"):
        mq.quantize(x[:, :40], **kw)
    with pytest.raises(ValueError, match="bfloat16, float16 or float32"):
        mq.quantize(x.to(torch.int32), **kw)
    with pytest.raises(ValueError, match="float32"):
        mq.dequantize(w, s, dtype=torch.float64, **kw)
    with pytest.raises(NotImplementedError, match="scales' dtype"):
        mq.dequantize(w, s.bfloat16(), s.bfloat16(), group_size=32, dtype=torch.float32)
    bank = _w(E=3)
    with pytest.raises(ValueError, match="batch dim"):
        mq.gather_qmm(x, w, s, **kw)
    with pytest.raises(ValueError, match="broadcast"):
        mq.gather_qmm(x[:, None], *bank, rhs_indices=torch.zeros(3, dtype=torch.int32), **kw)
    with pytest.raises(ValueError, match="integers"):
        mq.gather_qmm(x[:, None], *bank, rhs_indices=torch.zeros(4), **kw)


def test_empty_results(on_cpu):
    w, s = _w()
    x = torch.zeros(0, 256, dtype=torch.bfloat16)
    assert mq.quantized_matmul(x, w, s, mode="mxfp4").shape == (0, 48)
    assert mq.qqmm(x[None], w[:0], s[:0]).shape == (1, 0, 0)
    assert mq.quantize(x, mode="mxfp4")[1].shape == (0, 8)
    assert mq.dequantize(w[:0], s[:0], mode="mxfp4").shape == (0, 256)
    bank = _w(E=3)
    idx = torch.zeros(0, 2, dtype=torch.int32)
    out = mq.gather_qmm(x.reshape(0, 1, 1, 256), *bank, rhs_indices=idx, mode="mxfp4")
    assert out.shape == (0, 2, 1, 48)


def test_cpu_tensors_are_refused():
    w, s = _w()
    with pytest.raises(ValueError, match="GPU only"):
        mq.quantized_matmul(torch.zeros(1, 256, dtype=torch.bfloat16), w, s, mode="mxfp4")


def test_modules_hold_the_format():
    w, s = _w()
    lin = nn.QuantizedLinear(w, s, None, mode="mxfp4")
    assert (lin.input_dims, lin.output_dims, lin.group_size, lin.bits) == (256, 48, 32, 4)
    assert nn.QuantizedSwitchLinear(*_w(E=3), None, mode="mxfp4").num_experts == 3
    with pytest.raises(ValueError, match="no biases"):
        nn.QuantizedLinear(w, s, s, mode="mxfp4")
    with pytest.raises(ValueError, match="groups of 32"):
        nn.QuantizedLinear(w, s, None, group_size=64, mode="mxfp4")
    with pytest.raises(NotImplementedError):
        nn.QQLinear(w, s, mode="affine")
    # routing keeps the 4-bit-activation product of a QQLinear
    model = torch.nn.Sequential(nn.QQLinear(w, s), lin)
    dispatch.enable(model)
    assert type(model[0]) is nn.QQLinear and type(model[1]) is dispatch.DispatchedQuantizedLinear
    assert nn.QQLinear.forward is not nn.QuantizedLinear.forward


def test_checkpoint_modes(tmp_path):
    from safetensors.torch import save_file
    w, s = _w()
    b16 = torch.zeros(48, 4, dtype=torch.bfloat16)
    save_file({"a.weight": w.view(torch.uint32), "a.scales": s,
               "e.weight": _w(E=2)[0].view(torch.uint32), "e.scales": _w(E=2)[1],
               "h.weight": torch.zeros(48, 64, dtype=torch.int32).view(torch.uint32),
               "h.scales": b16, "h.biases": b16.clone()}, str(tmp_path / "model.safetensors"))
    cfg = {"quantization": {"group_size": 32, "bits": 4, "mode": "mxfp4",
                            "h": {"group_size": 64, "bits": 8}}}
    (tmp_path / "config.json").write_text(json.dumps(cfg))
    layers = checkpoint.quantized_layers(str(tmp_path), device="cpu")
    assert layers["a"].mode == layers["e"].mode == "mxfp4" and layers["a"].biases is None
    assert layers["a"].scales.dtype == torch.uint8
    assert (layers["h"].mode, layers["h"].bits, layers["h"].group_size) == ("affine", 8, 64)
    assert checkpoint.quant_params({"quantization": {"mode": "mxfp4"}}, "a", 32, 8) == (
        32, 4, "mxfp4")
    assert checkpoint.quant_params({"quantization": {"a": {"mode": "mxfp4"}}}, "a", 32, 8) == (
        32, 4, "mxfp4")


def test_rebit_spec():
    assert rebit.parse("attn=mxfp4,head=8") == {"attn": (4, 32, "mxfp4"), "head": (8, 64)}
    with pytest.raises(ValueError, match="32 only"):
        rebit.parse("attn=mxfp4:64")

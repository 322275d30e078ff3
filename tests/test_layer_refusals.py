"""Refusals of ca_rms_norm, ca_linear_q8, ca_gated_linear and ca_sample:
arguments are checked before anything is launched, so no GPU is needed."""
import ctypes

import pytest
import torch

import canvas_attn as ca
from canvas_attn import denoise as dn
from canvas_attn import layer

FAKE = 1 << 40  # an aligned address nothing reads
INV, UNS = ca.CA_ERR_INVALID, ca.CA_ERR_UNSUPPORTED


def call(fn, cls, base, kw):
    a = cls(**{**base, **kw})
    return fn(ctypes.byref(a), None)


NORM = dict(x=FAKE, x_type=0, w=FAKE, norm=1, eps=1e-6, out=FAKE, out_type=0, rows=3, cols=64)


@pytest.mark.parametrize("kw,status", [
    (dict(x=None), INV), (dict(out=None), INV), (dict(rows=-1), INV), (dict(cols=0), INV),
    (dict(x_type=2), INV), (dict(x_type=7), INV), (dict(out_type=3), INV), (dict(out_type=-1), INV),
    (dict(residual=FAKE), INV), (dict(sum_out=FAKE), INV),
    (dict(residual=FAKE, sum_out=FAKE, residual_type=2), INV), (dict(out_type=2), INV),
    (dict(eps=-1.0), INV), (dict(eps=float("nan")), INV), (dict(x_stride=63), INV),
    (dict(out_stride=63), INV), (dict(x=FAKE + 1), INV), (dict(w=FAKE + 2), INV),
    (dict(cols=1 << 31), UNS), (dict(rows=0), ca.CA_OK),
    (dict(rows=0, x=None, out=None), ca.CA_OK),
])
def test_rms_norm(kw, status):
    assert call(ca.lib.ca_rms_norm, layer.CaRmsNormArgs, NORM, kw) == status


LINEAR = dict(act=FAKE, act_scale=FAKE, w=FAKE, w_scale=FAKE, out=FAKE, n=2, rows=32, cols=64)
PRODUCT = [
    (dict(act=None), INV), (dict(out=None), INV), (dict(n=-1), INV), (dict(rows=0), INV),
    (dict(cols=0), INV), (dict(act=FAKE + 8), INV), (dict(out=FAKE + 1), INV),
    (dict(act_stride=48), INV), (dict(act_stride=65), INV), (dict(out_stride=31), INV),
    (dict(cols=68, act_stride=80), UNS), (dict(rows=1 << 31), UNS), (dict(n=1 << 31), UNS),
    (dict(n=0), ca.CA_OK), (dict(n=0, act=None, out=None), ca.CA_OK),
]


@pytest.mark.parametrize("kw,status", PRODUCT + [
    (dict(w=None), INV), (dict(w=FAKE + 4), INV), (dict(out=FAKE + 2, out_f32=1), INV),
    (dict(residual=FAKE, residual_stride=31), INV), (dict(residual=FAKE + 1), INV)])
def test_linear_q8(kw, status):
    assert call(ca.lib.ca_linear_q8, layer.CaLinearQ8Args, LINEAR, kw) == status


GATED = dict(act=FAKE, type=2, w_gate=FAKE, w_up=FAKE, out=FAKE, n=2, rows=32, cols=64)


@pytest.mark.parametrize("kw,status", PRODUCT + [
    (dict(w_gate=None), INV), (dict(w_up=None), INV), (dict(w_up=FAKE + 4), INV),
    (dict(type=1), INV), (dict(type=5), INV), (dict(activation=2), INV),
    (dict(activation=-1), INV), (dict(type=0, act_scale=FAKE), INV),
    (dict(type=0, up_scale=FAKE), INV), (dict(type=0, cols=60, act_stride=64), UNS)])
def test_gated_linear(kw, status):
    assert call(ca.lib.ca_gated_linear, layer.CaGatedLinearArgs, GATED, kw) == status


SAMPLE = dict(logits=FAKE, n_rows=4, n_vocab=100, n_cand=2, mask_id=-1, u=FAKE, temperature=1.0,
              top_p=1.0, token=FAKE)


@pytest.mark.parametrize("kw,status", [
    (dict(logits=None), INV), (dict(u=None), INV), (dict(token=None), INV), (dict(n_cand=-1), INV),
    (dict(n_vocab=0), INV), (dict(n_rows=-1), INV), (dict(n_suppress=-1), INV),
    (dict(n_suppress=2), INV), (dict(row_stride=99), INV), (dict(n_cand=5), INV),
    (dict(logits=FAKE + 2), INV), (dict(logits=FAKE + 1, logits_bf16=1), INV),
    (dict(n_vocab=376833), UNS), (dict(n_vocab=753665, logits_bf16=1), UNS),
    (dict(n_vocab=1 << 32), UNS), (dict(n_cand=0), ca.CA_OK),
    (dict(n_cand=0, logits=None, u=None, token=None), ca.CA_OK),
])
def test_sample(kw, status):
    assert call(ca.lib.ca_sample, dn.CaSampleArgs, SAMPLE, kw) == status


def test_null_arguments():
    for f in (ca.lib.ca_rms_norm, ca.lib.ca_linear_q8, ca.lib.ca_gated_linear, ca.lib.ca_sample):
        assert f(None, None) == INV


def z(*shape, t=torch.bfloat16):
    return torch.zeros(*shape).to(t)


F8, F32, I32 = torch.float8_e4m3fn, torch.float32, torch.int32


@pytest.mark.parametrize("make", [
    lambda: layer.make_rms_norm_args(z(2, 8, t=torch.float16), z(2, 8)),
    lambda: layer.make_rms_norm_args(z(2, 8), z(2, 9)),
    lambda: layer.make_rms_norm_args(z(2, 8), z(2, 8, t=F8)),
    lambda: layer.make_rms_norm_args(z(2, 8).T, z(8, 2)),
    lambda: layer.make_rms_norm_args(z(2, 8), z(2, 8), w=z(8)),
    lambda: layer.make_rms_norm_args(z(2, 8), z(2, 8), w=z(7, t=F32)),
    lambda: layer.make_rms_norm_args(z(2, 8), z(2, 8), sum_out=z(2, 8)),
    lambda: layer.make_rms_norm_args(z(2, 8), z(2, 8), residual=z(2, 8), sum_out=z(2, 8, t=F32)),
    lambda: layer.make_rms_norm_args(z(2, 8), z(2, 8, t=F8), out_scale=z(3, t=F32)),
    lambda: layer.make_linear_q8_args(z(2, 32), None, z(4, 32, t=F8), None, z(2, 4)),
    lambda: layer.make_linear_q8_args(z(2, 32, t=F8), None, z(4, 48, t=F8), None, z(2, 4)),
    lambda: layer.make_linear_q8_args(z(2, 32, t=F8), z(3, t=F32), z(4, 32, t=F8), None, z(2, 4)),
    lambda: layer.make_linear_q8_args(z(2, 32, t=F8), None, z(4, 32, t=F8), None, z(2, 5)),
    lambda: layer.make_linear_q8_args(z(2, 32, t=F8), None, z(4, 32, t=F8), None, z(2, 4),
                                      residual=z(2, 4, t=F32)),
    lambda: layer.make_gated_linear_args(z(2, 32), z(4, 32), z(4, 32, t=F8), z(2, 4)),
    lambda: layer.make_gated_linear_args(z(2, 32), z(4, 32), z(5, 32), z(2, 4)),
    lambda: layer.make_gated_linear_args(z(2, 32), z(4, 32), z(4, 32), z(2, 4), activation="relu"),
    lambda: layer.make_gated_linear_args(z(2, 32), z(4, 32), z(4, 32), z(2, 4),
                                         act_scale=z(2, t=F32)),
    lambda: layer.make_rms_norm_args(z(1, 8).expand(4, 8), z(4, 8)),
    lambda: layer.make_rms_norm_args(z(4, 8), z(1, 8).expand(4, 8)),
    lambda: layer.make_linear_q8_args(z(1, 32, t=F8).expand(2, 32), None, z(4, 32, t=F8), None,
                                      z(2, 4)),
    lambda: dn.make_sample_args(z(1, 9).expand(2, 9), None, z(2, t=F32), z(2, t=I32)),
    lambda: dn.make_sample_args(z(2, 9, t=torch.float16), None, z(2, t=F32), z(2, t=I32)),
    lambda: dn.make_sample_args(z(2, 9), None, z(3, t=F32), z(2, t=I32)),
    lambda: dn.make_sample_args(z(2, 9), None, z(3, t=F32), z(3, t=I32)),
    lambda: dn.make_sample_args(z(2, 9), None, z(2, t=F32), z(2, t=torch.int64)),
    lambda: dn.make_sample_args(z(2, 9), None, z(2, t=F32), z(2, t=I32), n_vocab=10),
    lambda: dn.make_sample_args(z(2, 9), None, z(2, t=F32), z(2, t=I32), top_k=z(2, t=F32)),
    lambda: dn.make_sample_args(z(2, 9), None, z(2, t=F32), z(2, t=I32), top_p=z(3, t=F32)),
])
def test_python_arguments(make):
    with pytest.raises(ValueError):
        make()


OFF = FAKE + 2  # 4-byte vectors that start between two entries


@pytest.mark.parametrize("name", ["act_scale", "w_scale", "bias", "status"])
def test_linear_q8_misaligned_vectors(name):
    assert call(ca.lib.ca_linear_q8, layer.CaLinearQ8Args, LINEAR, {name: OFF}) == INV


@pytest.mark.parametrize("name", ["act_scale", "gate_scale", "up_scale", "status"])
def test_gated_linear_misaligned_vectors(name):
    assert call(ca.lib.ca_gated_linear, layer.CaGatedLinearArgs, GATED, {name: OFF}) == INV


@pytest.mark.parametrize("name", ["rows", "u", "token", "prob", "temperature_row", "top_k_row",
                                  "top_p_row", "min_p_row", "suppress"])
def test_sample_misaligned_vectors(name):
    assert call(ca.lib.ca_sample, dn.CaSampleArgs, SAMPLE,
                {name: OFF, "n_suppress": int(name == "suppress")}) == INV


@pytest.mark.parametrize("make", [
    lambda: layer.make_rms_norm_args(z(2, 8), z(2, 8)),
    lambda: layer.make_linear_q8_args(z(2, 32, t=F8), None, z(4, 32, t=F8), None, z(2, 4)),
    lambda: layer.make_gated_linear_args(z(2, 32), z(4, 32), z(4, 32), z(2, 4)),
    lambda: dn.make_sample_args(z(2, 9, t=F32), None, z(2, t=F32), z(2, t=I32)),
])
def test_host_tensors_where_there_is_a_gpu(make, monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_available", lambda: False)
    make()
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    with pytest.raises(ValueError, match="cpu"):
        make()


@pytest.mark.parametrize("status", [z(1, t=F32), z(0, t=I32)])
def test_status_type(status):
    with pytest.raises(ValueError, match="status"):
        layer.make_linear_q8_args(z(2, 32, t=F8), None, z(4, 32, t=F8), None, z(2, 4),
                                  status=status)
    with pytest.raises(ValueError, match="status"):
        layer.make_gated_linear_args(z(2, 32), z(4, 32), z(4, 32), z(2, 4), status=status)

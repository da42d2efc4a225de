"""64-bit and bit-level references of the 4-bit cache and packed prompts.

The rounding points of a 4-bit row (rotated keys in f32, the scale in fp16)
are part of its definition, so its codes are compared exactly; everything
else is compared with the formulas in 64 bits.
"""
import ctypes

import numpy as np
import torch

from qx_b200 import BF16, F16, F32, MODEL_QWEN3
from qx_b200.runtime import model_shape

TORCH = {F32: torch.float32, BF16: torch.bfloat16, F16: torch.float16}
#: Half a step of each output type, relative to the value.
HALF_STEP = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}
SCALE = {0: 1.0 / 64.0, MODEL_QWEN3: 1.0 / np.sqrt(128.0)}

_libm = ctypes.CDLL("libm.so.6")
for _f in ("cosf", "sinf"):
    getattr(_libm, _f).restype = ctypes.c_float
    getattr(_libm, _f).argtypes = [ctypes.c_float]


def frequencies(model):
    """The f32 inverse frequencies of a model's rotation."""
    d = model_shape(model)[2]
    theta = 1e6 if model == MODEL_QWEN3 else 1e4
    return np.array([theta ** (-2.0 * i / d) for i in range(d // 2)], np.float64).astype(np.float32)


def angles(model, positions):
    return np.asarray(positions, np.float32)[:, None] * frequencies(model)


def rotate64(model, x, positions, norm=None):
    """Norm (Qwen) and rotation in 64 bits of x [tokens, heads, D] (numpy)."""
    x = np.asarray(x, np.float64)
    half = x.shape[-1] // 2
    if model == MODEL_QWEN3:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-6)
        if norm is not None:
            x = x * np.asarray(norm, np.float64)
    a = angles(model, positions).astype(np.float64)[:, None, :]
    left, right = x[..., :half], x[..., half:]
    return np.concatenate([left * np.cos(a) - right * np.sin(a), right * np.cos(a) + left * np.sin(a)], -1)


def qwen_keys32(x, positions, norm=None):
    """Qwen keys as a row holds them before quantisation: f32, each operation rounded."""
    x = np.asarray(x, np.float32)
    half = x.shape[-1] // 2
    mean = (x.astype(np.float64) ** 2).mean(-1, keepdims=True)
    x = x * (1.0 / np.sqrt(mean + 1e-6)).astype(np.float32)
    if norm is not None:
        x = x * np.asarray(norm, np.float32)
    a = angles(MODEL_QWEN3, positions)
    cos = np.array([[_libm.cosf(float(v)) for v in r] for r in a], np.float32)[:, None, :]
    sin = np.array([[_libm.sinf(float(v)) for v in r] for r in a], np.float32)[:, None, :]
    left, right = x[..., :half], x[..., half:]
    return np.concatenate([left * cos - right * sin, right * cos + left * sin], -1)


def quantise(x):
    """Codes 0..14 [..., D] and fp16 scales [..., D / 32] of f32 rows."""
    g = np.asarray(x, np.float32).reshape(*x.shape[:-1], -1, 32)
    scales = (np.abs(g).max(-1) / np.float32(7.0)).astype(np.float16)
    s = scales.astype(np.float32)[..., None]
    with np.errstate(divide="ignore", invalid="ignore"):
        codes = np.where(s > 0, np.clip(np.rint(g / s), -7, 7), 0.0)
    return (codes.reshape(x.shape) + 7).astype(np.uint8), scales


def values(codes, scales):
    """What codes and scales stand for, exact in 64 bits."""
    c = codes.astype(np.float64).reshape(*scales.shape, 32) - 7.0
    return (c * scales.astype(np.float64)[..., None]).reshape(codes.shape)


def unpack_rows(model, raw, key):
    """Codes [rows, heads, D] (the value's code plus 7: 0..14) and scales
    [rows, heads, D / 32] of raw 288-byte rows, by the layout include/qxcuda.h
    states."""
    hkv, d = model_shape(model)[1:]
    ng = d // 32
    n = raw.shape[0]
    scales = np.ascontiguousarray(raw[:, 256:]).view(np.float16).reshape(n, hkv, ng)
    body = np.ascontiguousarray(raw[:, :256]).reshape(n, hkv, d // 2)
    codes = np.zeros((n, hkv, d), np.uint8)
    words = body.view(np.uint32).astype(np.int64)
    for dim in range(d):
        j, r = dim // 32, dim % 32
        if key:
            w = words[:, :, (r // 8) * ng + j] >> (8 * (r % 4) + (4 if r % 8 < 4 else 0))
            codes[:, :, dim] = ((w & 15) ^ 8) - 1  # two's complement plus 7
        else:
            nibble = 4 * ((r % 8) * ng + j) + r // 8
            codes[:, :, dim] = (body[:, :, nibble // 2] >> (4 * (nibble % 2))) & 15
    return codes, scales


def attend64(model, q, k, v):
    """Attention in 64 bits of q [Hq, D] over k, v [rows, Hkv, D], and the
    weighted mean of |v| (what relative errors of the weights multiply)."""
    hq, hkv, d = model_shape(model)
    q = torch.as_tensor(q, dtype=torch.float64).view(hkv, hq // hkv, d)
    k, v = (torch.as_tensor(x, dtype=torch.float64) for x in (k, v))
    p = torch.softmax(torch.einsum("hgd,thd->hgt", q, k) * SCALE[model], -1)
    out = torch.einsum("hgt,thd->hgd", p, v).reshape(hq, d)
    mean = torch.einsum("hgt,thd->hgd", p, v.abs()).reshape(hq, d)
    return out.numpy(), mean.numpy()


def logit_error(model, q, k, bits):
    """Bound of an f32 logit's error: |q|.|k| times `bits` roundings' worth."""
    hq, hkv, d = model_shape(model)
    q = np.abs(np.asarray(q, np.float64)).reshape(hkv, hq // hkv, d)
    top = np.abs(np.asarray(k, np.float64)).max(0)  # [Hkv, D]
    return float(np.einsum("hgd,hd->hg", q, top).max() * SCALE[model] * bits * 2.0 ** -24)


def close(actual, expected, tolerance):
    """max |actual - expected| / tolerance, elementwise (<= 1 passes)."""
    diff = np.abs(np.asarray(actual, np.float64) - expected)
    assert np.isfinite(diff).all()
    return float((diff / tolerance).max()) if diff.size else 0.0

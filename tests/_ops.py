"""Plain 64-bit forms of the row operators, and the types they come in."""
import numpy as np
import torch

U = 2.0 ** -24  # half a step of f32, relative
TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CODE = {"f32": 0, "bf16": 1, "f16": 2}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}  # half a step, relative
LEAST = {"f32": 2.0 ** -149, "bf16": 2.0 ** -133, "f16": 2.0 ** -25}  # half the least subnormal, at most


def stored(a, dtype):
    """f64 array -> (bytes as the device holds them, the f64 values they stand for)."""
    t = torch.from_numpy(np.ascontiguousarray(a, np.float64)).to(TORCH[dtype])
    return t.view(torch.uint8).numpy() if t.numel() else np.zeros(0, np.uint8), t.double().numpy()


def values(raw, dtype, shape):
    """Device bytes -> f64 values."""
    return torch.from_numpy(np.ascontiguousarray(raw).view(np.uint8).copy()).view(TORCH[dtype]).double().numpy().reshape(shape)


def e4m3(raw, shape):
    return torch.from_numpy(np.ascontiguousarray(raw).view(np.uint8).copy()).view(torch.float8_e4m3fn).double().numpy().reshape(shape)


def dev(oco, a):
    return oco.DeviceBuffer.from_array(np.ascontiguousarray(a))


def quantized(x, exact_operands):
    """(codes as bytes [rows, k], f32 scales [blocks, rows]) of f64 rows: the quotient 448 x / max|x| rounded to
    f32 once (exact_operands: from exact operands; else from f32(0.875 x) and f32(max / 512)), then to e4m3."""
    rows, k = x.shape
    codes, scales = np.zeros((rows, k), np.uint8), np.zeros((-(-k // 128), rows), np.float32)
    for b in range(len(scales)):
        part = x[:, 128 * b:128 * b + 128]
        top = np.maximum(np.abs(part).max(1), 448.0 * 2.0 ** -126)
        scales[b] = top.astype(np.float32) / np.float32(448.0)
        if exact_operands:
            q = (448.0 * part / top[:, None]).astype(np.float32)
        else:
            q = (part.astype(np.float32) * np.float32(0.875)) / (top.astype(np.float32) / np.float32(512.0))[:, None]
        codes[:, 128 * b:128 * b + 128] = torch.from_numpy(q).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    return codes, scales

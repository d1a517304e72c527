"""quantizeInt8 / matmulInt8 / groupRows / matmulInt8Grouped -- products in 8-bit integers.

The reference has block-quantized weights only (src/ops/quantize.js:71-118).  Here the weights have one
scale per channel and the activations one per token, and the product runs on the integer tensor cores:

    scale(x) = max|x| / 127           code(x)[k] = round-half-to-even(127 x[k] / max|x|)
    c[m, n]  = scale(a_m) scale(w_n) sum_k code(a_m)[k] code(w_n)[k]          (the sum is exact)

``quantizeInt8`` packs one matrix [K, N] or one per expert [E, K, N]; ``matmulInt8`` multiplies by one
matrix, ``matmulInt8Grouped`` each row by the matrix of its expert, with the lists ``groupRows`` makes.
Arguments, records and errors are in the manner of quantizeQ8 / matmulQ8; the direct, asynchronous forms
on device buffers, with row pitches, are device.int8Pack, int8Matmul, int8MatmulGrouped and groupRows.
"""
import numpy as np

from .. import device
from .. import tensor as T
from ..dispatch import run
from .matmul import _contiguous, k as kernelName
from .quantize import Quantized, _field


def _float(name, t):
    if t.dtype not in ("f32", "f16"):
        raise ValueError(f"{name}: f32 or f16 expected, got {t.dtype}")
    return _contiguous(t)


def quantizeInt8(weight):
    """Pack an f32 or f16 weight [K, N], or [E, K, N] with a matrix per expert, into 8-bit codes and a scale
    per channel.  The record {buffer, K, N, experts, totalBytes} is read by matmulInt8 / matmulInt8Grouped."""
    _float("quantizeInt8", weight)
    if len(weight.shape) not in (2, 3):
        raise ValueError(f"quantizeInt8: a weight [K, N] or [experts, K, N] expected, got {len(weight.shape)}D")
    experts = weight.shape[0] if len(weight.shape) == 3 else 1
    K, N = weight.shape[-2:]
    totalBytes = device.int8PackedBytes(K, N, experts)
    buffer = device.alloc(totalBytes, device.PRIVATE)
    try:
        run(kernelName("quantize_int8", weight.dtype), [
            {"buffer": weight.buffer, "index": 0},
            {"buffer": buffer, "index": 1},
        ], {"x": N, "y": K, "z": experts}, {"x": min(N, 256), "y": 1},
            {"data": np.array([K, N, experts], dtype=np.uint32), "index": 2})
    except Exception:
        device.releaseBuffer(buffer)
        raise
    return Quantized(buffer=buffer, K=K, N=N, experts=experts, totalBytes=totalBytes)


def matmulInt8(a, w):
    """C[M,N] = A[M,K](f32 or f16) @ W[K,N](int8 per channel), in A's type."""
    N, K, experts, wBuffer = (_field(w, f) for f in ("N", "K", "experts", "buffer"))
    _float("matmulInt8", a)
    if len(a.shape) != 2:
        raise ValueError(f"matmulInt8: activations [M, K] expected, got {len(a.shape)}D")
    if experts != 1:
        raise ValueError(f"matmulInt8: the weights hold {experts} experts; use matmulInt8Grouped")
    M = a.shape[0]
    if a.shape[1] != K:
        raise ValueError(f"matmulInt8: inner dims don't match: {a.shape[1]} vs {K}")
    out = T.create([M, N], a.dtype)
    run(kernelName("matmul_int8", a.dtype), [
        {"buffer": a.buffer, "index": 0},
        {"buffer": wBuffer, "index": 1},
        {"buffer": out.buffer, "index": 2},
    ], {"x": N, "y": M}, {"x": min(N, 16), "y": min(M, 16) or 1},
        {"data": np.array([M, N, K], dtype=np.uint32), "index": 3})
    return out


def groupRows(ids, experts):
    """Sort rows by expert: ids i32 [rows], or [tokens, top] with `top` experts per token; an id outside
    [0, experts) is a row of no expert.  The record {offsets, order, position, rows, experts, fan}:
    expert e's rows are the sorted places offsets[e] .. offsets[e + 1], order[j] is the row at place j
    (rows of one expert in their order, rows of no expert last), position is its inverse."""
    if ids.dtype != "i32":
        raise ValueError(f"groupRows: i32 ids expected, got {ids.dtype}")
    if len(ids.shape) not in (1, 2):
        raise ValueError(f"groupRows: ids [rows] or [tokens, top] expected, got {len(ids.shape)}D")
    _contiguous(ids)
    rows, experts = ids.size, int(experts)
    if not 1 <= experts <= 1024:
        raise ValueError(f"groupRows: 1 to 1024 experts are taken, got {experts}")
    fan = ids.shape[1] if len(ids.shape) == 2 else 1
    offsets, order, position = T.create([experts + 1], "i32"), T.create([rows], "i32"), T.create([rows], "i32")
    run("group_rows", [
        {"buffer": ids.buffer, "index": 0},
        {"buffer": offsets.buffer, "index": 1},
        {"buffer": order.buffer, "index": 2},
        {"buffer": position.buffer, "index": 3},
    ], {"x": max(rows, 1)}, None, {"data": np.array([rows, experts], dtype=np.uint32), "index": 4})
    return Quantized(offsets=offsets, order=order, position=position, rows=rows, experts=experts, fan=fan)


def matmulInt8Grouped(a, w, groups, gather=True, scatter=False):
    """Rows times the matrix of their expert.  ``groups`` is groupRows' record.  With ``gather`` A holds the
    groups.rows / groups.fan tokens, each of which goes to the places of its fan ids; without it the
    groups.rows rows in sorted order, as an earlier product left them.  The result [rows, N], in A's type,
    is in sorted order, or with ``scatter`` in the order of the ids; rows of no expert are zero."""
    N, K, experts, wBuffer = (_field(w, f) for f in ("N", "K", "experts", "buffer"))
    rows, fan = _field(groups, "rows"), _field(groups, "fan")
    _float("matmulInt8Grouped", a)
    if len(a.shape) != 2:
        raise ValueError(f"matmulInt8Grouped: activations [rows, K] expected, got {len(a.shape)}D")
    if experts != _field(groups, "experts"):
        raise ValueError(f"matmulInt8Grouped: {experts} experts in the weights, {_field(groups, 'experts')} in the groups")
    if a.shape[1] != K:
        raise ValueError(f"matmulInt8Grouped: inner dims don't match: {a.shape[1]} vs {K}")
    want = rows // fan if gather and fan else rows
    if a.shape[0] != want:
        raise ValueError(f"matmulInt8Grouped: {a.shape[0]} rows of activations, {want} expected")
    out = T.zeros([rows, N], a.dtype)
    buffers = [
        {"buffer": a.buffer, "index": 0},
        {"buffer": wBuffer, "index": 1},
        {"buffer": out.buffer, "index": 2},
        {"buffer": _field(groups, "offsets").buffer, "index": 4},
    ]
    if gather:
        buffers.append({"buffer": _field(groups, "position").buffer, "index": 5})
    if scatter:
        buffers.append({"buffer": _field(groups, "order").buffer, "index": 6})
    run(kernelName("matmul_int8_grouped", a.dtype), buffers, {"x": N, "y": max(rows, 1)},
        {"x": min(N, 16), "y": min(max(rows, 1), 16)},
        {"data": np.array([rows, N, K, experts, max(fan, 1)], dtype=np.uint32), "index": 3})
    return out

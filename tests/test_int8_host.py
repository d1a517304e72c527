"""The 8-bit integer products on the host side: messages, parameter checks and costs (no device)."""
import numpy as np
import pytest

import int8_reference as R
import smith_b200 as smith
from smith_b200 import device
from smith_b200 import profile as P


class _T:
    def __init__(self, shape, dtype="f32"):
        self.shape, self.dtype, self.buffer = list(shape), dtype, None
        self.strides, self.size = smith.tensor.computeStrides(shape), int(np.prod(shape))


def _record(K, N, experts=1):
    return {"buffer": None, "K": K, "N": N, "experts": experts, "totalBytes": 0}


def _groups(rows, experts, fan):
    return {"offsets": None, "order": None, "position": None, "rows": rows, "experts": experts, "fan": fan}


@pytest.mark.parametrize("call,text", [
    (lambda: smith.matmulInt8(_T([2, 48]), _record(64, 8)), "matmulInt8: inner dims don't match: 48 vs 64"),
    (lambda: smith.matmulInt8(_T([2, 64], "i32"), _record(64, 8)), "matmulInt8: f32 or f16 expected, got i32"),
    (lambda: smith.matmulInt8(_T([2, 2, 64]), _record(64, 8)), "matmulInt8: activations [M, K] expected, got 3D"),
    (lambda: smith.matmulInt8(_T([2, 64]), _record(64, 8, 3)),
     "matmulInt8: the weights hold 3 experts; use matmulInt8Grouped"),
    (lambda: smith.quantizeInt8(_T([64])), "quantizeInt8: a weight [K, N] or [experts, K, N] expected, got 1D"),
    (lambda: smith.quantizeInt8(_T([64, 8], "u8")), "quantizeInt8: f32 or f16 expected, got u8"),
    (lambda: smith.groupRows(_T([4, 2]), 8), "groupRows: i32 ids expected, got f32"),
    (lambda: smith.groupRows(_T([4, 2, 2], "i32"), 8), "groupRows: ids [rows] or [tokens, top] expected, got 3D"),
    (lambda: smith.groupRows(_T([4, 2], "i32"), 1025), "groupRows: 1 to 1024 experts are taken, got 1025"),
    (lambda: smith.groupRows(_T([4, 2], "i32"), 0), "groupRows: 1 to 1024 experts are taken, got 0"),
    (lambda: smith.matmulInt8Grouped(_T([4, 48]), _record(64, 8, 2), _groups(8, 2, 2)),
     "matmulInt8Grouped: inner dims don't match: 48 vs 64"),
    (lambda: smith.matmulInt8Grouped(_T([4, 64]), _record(64, 8, 3), _groups(8, 2, 2)),
     "matmulInt8Grouped: 3 experts in the weights, 2 in the groups"),
    (lambda: smith.matmulInt8Grouped(_T([5, 64]), _record(64, 8, 2), _groups(8, 2, 2)),
     "matmulInt8Grouped: 5 rows of activations, 4 expected"),
    (lambda: smith.matmulInt8Grouped(_T([4, 64]), _record(64, 8, 2), _groups(8, 2, 2), gather=False),
     "matmulInt8Grouped: 4 rows of activations, 8 expected"),
])
def test_messages(call, text):
    with pytest.raises(ValueError) as e:
        call()
    assert str(e.value) == text


def test_strided_tensors_are_refused():
    t = _T([4, 64])
    t.strides = [128, 1]
    with pytest.raises(ValueError, match="contiguous"):
        smith.matmulInt8(t, _record(64, 8))


def test_packed_size_and_its_limits():
    """Whole tiles of 128 channels by 128 k, and a maximum per channel of a tile."""
    for K, N, E in [(1, 1, 1), (128, 128, 1), (129, 128, 1), (128, 129, 3), (4096, 14336, 1), (131072, 4, 1024)]:
        nt, ks = -(-N // 128), -(-K // 128)
        assert device.int8PackedBytes(K, N, E) == E * nt * (ks * 128 * 128 + 128 * 4)
    for K, N, E in [(0, 1, 1), (131073, 1, 1), (1, 0, 1), (1, (1 << 22) + 1, 1), (1, 1, 0), (1, 1, 1025)]:
        with pytest.raises(device.SmithError):
            device.int8PackedBytes(K, N, E)


def test_costs():
    assert P.algorithmicCost("matmul_int8", [16, 100, 64]) == (4 * (16 * 64 + 16 * 100) + 100 * 68, 2 * 16 * 64 * 100)
    assert P.algorithmicCost("matmul_int8_f16", [16, 100, 64]) == (2 * (16 * 64 + 16 * 100) + 100 * 68, 2 * 16 * 64 * 100)
    assert P.algorithmicCost("matmul_int8_grouped", [16, 100, 64, 5, 2]) == (
        4 * (8 * 64 + 16 * 100) + 5 * 100 * 68, 2 * 16 * 64 * 100)
    assert P.algorithmicCost("quantize_int8", [64, 100, 2]) == (2 * 100 * (4 * 64 + 64 + 4), 0)
    assert P.algorithmicCost("group_rows", [64, 5]) == (4 * (3 * 64 + 6), 0)


def test_unknown_checkpoint_kind(tmp_path):
    with pytest.raises(ValueError, match="'i8'"):
        smith.saveQuantized({"x": ("q5", {"totalBytes": 0, "groups": 0, "N": 0})}, str(tmp_path / "x"))


def test_reference_codes_by_hand():
    c, s = R.codes(np.array([[254, 1, 3, -1, -3, 5, 0]], np.float32), 1)
    assert c.tolist() == [[127, 0, 2, 0, -2, 2, 0]] and s[0] == 254
    c, s = R.codes(np.array([[0, 0], [np.inf, 1], [np.nan, 1]], np.float32), 1)
    assert not c.any() and s[0] == 0 and np.isnan(s[1:]).all()
    offsets, order, position = R.group_rows([2, -1, 0, 2, 5], 3)
    assert offsets.tolist() == [0, 1, 1, 3] and order.tolist() == [2, 0, 3, 1, 4] and position.tolist() == [1, 3, 0, 2, 4]

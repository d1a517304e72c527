"""-m gpu: the 8-bit integer products, the ragged form by expert and the sort that feeds it.

The sums are whole numbers and exact, and the definition names the order of the f32 operations that
follow, so every comparison here is bit for bit (tests/int8_reference.py); there are no tolerances.
"""
import numpy as np
import pytest

import int8_reference as R
import smith_b200 as smith
from gpu_util import DevBuf
from smith_b200 import device

pytestmark = pytest.mark.gpu
DTYPE = {np.float32: device.DTYPE_F32, np.float16: device.DTYPE_F16}


def dt(array):
    return device.DTYPE_F16 if array.dtype == np.float16 else device.DTYPE_F32


def pack(w):
    w3 = w if w.ndim == 3 else w[None]
    E, K, N = w3.shape
    wb, out = DevBuf.of(w3), DevBuf(device.int8PackedBytes(K, N, E))
    device.int8Pack(dt(w), wb.handle, out.handle, K, N, E)
    device.synchronize()
    wb.free()
    return out


def matmul(a, packed, N, lda=0, ldc=0):
    """a: the values in rows of lda; returns whole C rows of ldc, what no output fills keeping NaN."""
    M, K = a.shape
    wide = np.zeros((M, lda or K), a.dtype)
    wide[:, :K] = a
    wide[:, K:] = np.nan                              # what lies between the rows is not read
    ab, cb = DevBuf.of(wide), DevBuf.of(np.full((M, ldc or N), np.nan, a.dtype))
    device.int8Matmul(dt(a), ab.handle, packed.handle, cb.handle, M, N, K, lda, ldc)
    device.synchronize()
    assert device.kernelStatus() == 0, "a bounded device-side wait gave up"
    return cb.get(a.dtype).reshape(M, ldc or N)


def data(seed, M, K, N, dtype, experts=None):
    rng = np.random.default_rng(seed)
    a = (rng.standard_normal((M, K)) * rng.uniform(0.1, 5, (M, 1))).astype(dtype)
    shape = (K, N) if experts is None else (experts, K, N)
    return a, (rng.standard_normal(shape) * rng.uniform(0.5, 2, (1, N)) / np.sqrt(K)).astype(dtype)


# one value; one tile; sizes off every tile in all directions; one token and few tokens on long and wide
# weights; token counts either side of every tile size; many tiles
SHAPES = [(1, 1, 1), (1, 2, 3), (2, 33, 5), (1, 128, 128), (16, 128, 128), (17, 127, 129), (15, 129, 257), (1, 4096, 1024),
          (4, 14336, 136), (8, 640, 4096), (31, 1000, 300), (32, 1024, 512), (33, 384, 640), (63, 100, 1000),
          (64, 2048, 130), (65, 257, 513), (127, 513, 255), (128, 512, 512), (129, 511, 513), (255, 640, 384),
          (256, 256, 256), (257, 1100, 300), (511, 384, 1000), (513, 2048, 640), (700, 130, 2000), (1031, 900, 777),
          (200, 20001, 300), (150, 64, 20000), (4097, 128, 128), (2500, 1024, 2500), (16, 14336, 4096), (100, 5000, 24)]


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_product_is_the_definition_bit_for_bit(M, K, N, dtype):
    a, w = data(M * 7 + K, M, K, N, dtype)
    got = matmul(a, pack(w), N)
    assert R.same_bits(got, R.product(a, w))


@pytest.mark.parametrize("wide", [1, 3, 8, 24])
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_row_pitches(dtype, wide):
    """Rows of A and C inside wider ones: what lies between is neither read nor written."""
    for M, K, N in [(5, 300, 70), (130, 257, 200)]:
        a, w = data(3, M, K, N, dtype)
        got = matmul(a, pack(w), N, K + wide, N + 2 * wide + 1)
        assert R.same_bits(np.ascontiguousarray(got[:, :N]), R.product(a, w))
        assert np.isnan(got[:, N:]).all()


@pytest.mark.parametrize("M", [3, 40, 300])
def test_ties_round_to_even(M):
    """max = 254 and whole values: 127 x / 254 = x / 2, every odd value on the border of two codes."""
    rng = np.random.default_rng(M)
    a = rng.integers(-254, 255, (M, 200)).astype(np.float32)
    w = rng.integers(-254, 255, (200, 150)).astype(np.float32)
    a[:, 7], w[9] = 254, -254
    assert R.same_bits(matmul(a, pack(w), 150), R.product(a, w))
    assert R.same_bits(matmul(a.astype(np.float16), pack(w.astype(np.float16)), 150),
                       R.product(a.astype(np.float16), w.astype(np.float16)))


def test_values_next_to_a_border():
    """Neighbours, in f32, of the values where 127 x / max crosses from one code to the next."""
    rng = np.random.default_rng(0)
    a = np.empty((64, 3 * 254 + 1), np.float32)
    for r in range(64):
        most = np.float32(np.exp(rng.uniform(-60, 60)))
        half = (np.arange(-127, 127) + 0.5) / 127 * float(most)
        near = half.astype(np.float32)
        a[r] = np.concatenate([[most], near, np.nextafter(near, np.float32(np.inf)), np.nextafter(near, np.float32(-np.inf))])
    w = np.eye(a.shape[1], dtype=np.float32)                      # each output is one code: nothing averages out
    assert R.same_bits(matmul(a, pack(w), w.shape[1]), R.product(a, w))
    assert R.same_bits(matmul(w, pack(np.ascontiguousarray(a.T)), 64), R.product(w, a.T))


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_extraordinary_rows_and_channels(dtype):
    """Zeros, infinities, NaNs, the smallest and the largest values: each stays in its row and channel."""
    M, K, N = 40, 260, 140
    a, w = data(11, M, K, N, dtype)
    big, tiny = np.finfo(dtype).max, np.finfo(dtype).smallest_subnormal
    a[0] = 0
    a[1, 5], a[2, 6], a[3, 7] = np.inf, -np.inf, np.nan
    a[4] = tiny
    a[5] = tiny * np.arange(K, dtype=np.float64).astype(dtype)
    a[6, 0] = big
    a[7, -1] = np.nan
    a[8] *= dtype(1e-4)
    w[:, 0] = 0
    w[3, 1], w[-1, 2], w[0, 139] = np.inf, np.nan, -np.inf
    w[:, 4] = tiny
    w[:, 5] = big
    got, want = matmul(a, pack(w), N), R.product(a, w)
    assert R.same_bits(got, want)
    assert np.isnan(got[[1, 2, 3, 7]]).all() and np.isnan(got[:, [1, 2, 139]]).all()
    others = np.delete(np.delete(got, [1, 2, 3, 7], 0), [1, 2, 139], 1)
    assert not np.isnan(others).any()


def test_longest_reduction_is_exact():
    """K = 131072 with codes of 127 throughout: the sum 127^2 K is just below 2^31."""
    K, N = 131072, 130
    a, w = np.ones((3, K), np.float32), np.ones((K, N), np.float32)
    a[1] = -1
    a[2, ::2] = -1
    got = matmul(a, pack(w), N)
    assert R.same_bits(got, R.product(a, w))
    assert got[0, 0] == pytest.approx(K, rel=1e-6) and got[2, 0] == 0


def test_result_may_take_the_place_of_the_activations():
    a, w = data(5, 70, 256, 256, np.float32)
    packed, ab = pack(w), DevBuf.of(a)
    device.int8Matmul(device.DTYPE_F32, ab.handle, packed.handle, ab.handle, 70, 256, 256)
    device.synchronize()
    assert R.same_bits(ab.get(np.float32).reshape(70, 256), R.product(a, w))


def test_offsets_beyond_32_bits():
    """Rows of A further than 4 GB apart, and a C of more than 2^31 values."""
    K, N = 200, 96
    a, w = data(6, 3, K, N, np.float16)
    packed, lda = pack(w), (1 << 30) + 8
    ab = DevBuf((2 * lda + K) * 2)
    for r in range(3):
        device.upload(ab.handle, a[r], offset=2 * r * lda)
    cb = DevBuf(3 * N * 2)
    device.int8Matmul(device.DTYPE_F16, ab.handle, packed.handle, cb.handle, 3, N, K, lda)
    device.synchronize()
    assert R.same_bits(cb.get(np.float16).reshape(3, N), R.product(a, w))
    ab.free()
    ldc = (1 << 30) + 8
    cb = DevBuf((2 * ldc + N) * 2)
    ab = DevBuf.of(a)
    device.int8Matmul(device.DTYPE_F16, ab.handle, packed.handle, cb.handle, 3, N, K, 0, ldc)
    device.synchronize()
    got = np.stack([device.download(cb.handle, N * 2, np.float16, offset=2 * r * ldc) for r in range(3)])
    assert R.same_bits(got, R.product(a, w))
    cb.free()


# ------------------------------------------------------------------------------------------ by expert

def grouped(a, packed, offsets, rows, N, K, E, position=None, order=None, fan=1, fill=np.nan, lda=0, ldc=0):
    ab, ob = DevBuf.of(a), DevBuf.of(np.asarray(offsets, np.int32))
    pb = None if position is None else DevBuf.of(np.asarray(position, np.int32))
    rb = None if order is None else DevBuf.of(np.asarray(order, np.int32))
    width = ldc or N
    guard = 64                                                    # values before and after that nothing may touch
    cb = DevBuf.of(np.full(rows * width + 2 * guard, fill, a.dtype))
    inner = device.wrapDeviceMemory(device.devicePtr(cb.handle) + guard * a.itemsize, rows * width * a.itemsize)
    device.int8MatmulGrouped(dt(a), ab.handle, packed.handle, ob.handle, inner, rows, N, K, E, lda, ldc,
                             pb and pb.handle, rb and rb.handle, fan)
    device.synchronize()
    assert device.kernelStatus() == 0, "a bounded device-side wait gave up"
    device.releaseBuffer(inner)
    whole = cb.get(a.dtype)
    assert R.same_bits(whole[:guard], np.full(guard, fill, a.dtype)) and R.same_bits(whole[-guard:], np.full(guard, fill, a.dtype))
    return whole[guard:-guard].reshape(rows, width)


def expected(a_sorted, w, offsets, order=None, fill=np.nan):
    """a_sorted: activations per sorted place."""
    rows, N = a_sorted.shape[0], w.shape[2]
    c = np.full((rows, N), fill, a_sorted.dtype)
    for e in range(w.shape[0]):
        at = np.arange(offsets[e], offsets[e + 1])
        if at.size:
            c[at if order is None else order[at]] = R.product(a_sorted[at], w[e])
    return c


GROUPED = [  # tokens, fan, experts, K, N
    (1, 1, 1, 64, 64), (1, 8, 16, 300, 200), (3, 2, 5, 128, 128), (16, 2, 8, 257, 130), (40, 4, 64, 200, 70),
    (150, 2, 3, 640, 300), (301, 2, 12, 131, 277), (64, 8, 1024, 40, 20), (700, 1, 2, 100, 513), (513, 4, 9, 384, 256), (3000, 2, 4, 1300, 520), (40000, 4, 1024, 64, 40),
    (5, 100, 7, 90, 33), (2, 8, 8, 4096, 1024)]


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("T,fan,E,K,N", GROUPED)
def test_grouped_product(T, fan, E, K, N, dtype):
    """Uneven groups, some empty, some rows of no expert; tokens gathered and results put back."""
    rng = np.random.default_rng(T + E)
    share = rng.dirichlet(np.full(E, 0.3))
    ids = rng.choice(E, size=(T, fan), p=share).astype(np.int32)
    ids[rng.random((T, fan)) < 0.1] = -1
    offsets, order, position = R.group_rows(ids, E)
    rows = T * fan
    a, w = data(T, T, K, N, dtype, experts=E)
    packed = pack(w)
    a_sorted = a[order // fan]
    up = grouped(a, packed, offsets, rows, N, K, E, position, None, fan)
    assert R.same_bits(up, expected(a_sorted, w, offsets))
    down = grouped(np.ascontiguousarray(a_sorted), packed, offsets, rows, N, K, E, None, order)
    assert R.same_bits(down, expected(a_sorted, w, offsets, order))
    both = grouped(a, packed, offsets, rows, N, K, E, position, order, fan, ldc=N + 3)
    assert R.same_bits(np.ascontiguousarray(both[:, :N]), expected(a_sorted, w, offsets, order))
    assert np.isnan(both[:, N:]).all()


@pytest.mark.parametrize("sizes", [[0, 0, 0, 0], [0, 50, 0, 0], [300, 0, 0, 1], [0, 0, 0, 257], [16, 16, 16, 16], [1, 1, 1, 1],
                                   [31, 33, 128, 129]])
def test_group_sizes(sizes):
    """No rows at all, one group with everything, groups at and around the tile sizes, rows behind the last."""
    E, K, N, behind = 4, 150, 260, 21
    rows = sum(sizes) + behind
    offsets = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
    a, w = data(sum(sizes), rows, K, N, np.float32, experts=E)
    got = grouped(a, pack(w), offsets, rows, N, K, E)
    assert R.same_bits(got, expected(a, w, offsets))
    assert np.isnan(got[sum(sizes):]).all()


def test_lists_that_lead_outside_are_skipped():
    """Places, rows and boundaries outside the arrays touch nothing and leave the other rows right."""
    E, K, N, rows = 3, 90, 100, 60
    offsets, order = np.array([0, 20, 40, 60], np.int32), np.arange(rows, dtype=np.int32)[::-1].copy()
    a, w = data(2, rows, K, N, np.float32, experts=E)
    packed = pack(w)
    bad = order.copy()
    bad[[0, 21, 59]] = [-1, rows, 2 ** 31 - 1]
    want = expected(a, w, offsets, order)
    want[order[[0, 21, 59]]] = np.nan
    assert R.same_bits(grouped(a, packed, offsets, rows, N, K, E, None, bad), want)
    place = np.arange(rows, dtype=np.int32)
    place[[5, 30]] = [-7, rows + 100]                             # sorted places 5 and 30 then hold anything
    got = grouped(a, packed, offsets, rows, N, K, E, place, None)
    keep = np.delete(np.arange(rows), [5, 30])
    assert R.same_bits(got[keep], expected(a, w, offsets)[keep])
    for wild in ([-5, 20, 40, 1000], [0, 2 ** 31 - 1, -2 ** 31, 60], [60, 40, 20, 0], [70, 80, 90, 100]):
        grouped(a, packed, np.array(wild, np.int32), rows, N, K, E)          # stays inside C
    got = grouped(a, packed, np.array([-5, 20, 40, 1000], np.int32), rows, N, K, E)
    assert R.same_bits(got, expected(a, w, offsets))


def sort_on_device(ids, E):
    ids = np.asarray(ids, np.int32)
    n = ids.size
    ib = DevBuf.of(ids)
    outs = [DevBuf.of(np.full(max(m, 1), -77, np.int32)) for m in (E + 1, n, n)]
    device.groupRows(ib.handle, *(o.handle for o in outs), n, E)
    device.synchronize()
    return [o.get(np.int32)[:m] for o, m in zip(outs, (E + 1, n, n))]


@pytest.mark.parametrize("E", [1, 2, 7, 32, 256, 1023, 1024])
@pytest.mark.parametrize("n", [0, 1, 31, 32, 33, 500, 4096, 4097, 20011])
def test_group_rows(n, E):
    rng = np.random.default_rng(n + E)
    for ids in (rng.integers(0, E, n), rng.integers(-2, E + 3, n), np.full(n, E - 1), np.full(n, -1),
                np.where(rng.random(n) < 0.01, -2 ** 31, 2 ** 31 - 1), np.sort(rng.integers(0, E, n))[::-1]):
        for got, want in zip(sort_on_device(ids, E), R.group_rows(ids, E)):
            assert np.array_equal(got, want)


def test_group_rows_large():
    ids = (np.random.default_rng(1).pareto(1.0, 1_000_003) * 20).astype(np.int64).clip(0, 300)
    for got, want in zip(sort_on_device(ids, 256), R.group_rows(ids, 256)):
        assert np.array_equal(got, want)


def test_a_run_together():
    """What an expert layer does: sort, the first product from tokens, the second back to the ids' order --
    without a word from the host in between."""
    T, fan, E, K, F = 77, 3, 6, 260, 390
    rng = np.random.default_rng(4)
    ids = np.stack([rng.permutation(E)[:fan] for _ in range(T)]).astype(np.int32)
    ids[70:] = -1
    a, w1 = data(1, T, K, F, np.float16, experts=E)
    _, w2 = data(2, T, F, K, np.float16, experts=E)
    rows = T * fan
    p1, p2, ab, ib = pack(w1), pack(w2), DevBuf.of(a), DevBuf.of(ids)
    lists = [DevBuf((E + 1) * 4), DevBuf(rows * 4), DevBuf(rows * 4)]
    hb, cb = DevBuf.of(np.zeros((rows, F), np.float16)), DevBuf.of(np.zeros((rows, K), np.float16))
    device.groupRows(ib.handle, *(x.handle for x in lists), rows, E)
    device.int8MatmulGrouped(device.DTYPE_F16, ab.handle, p1.handle, lists[0].handle, hb.handle, rows, F, K, E,
                             positionBuffer=lists[2].handle, fan=fan)
    device.int8MatmulGrouped(device.DTYPE_F16, hb.handle, p2.handle, lists[0].handle, cb.handle, rows, K, F, E,
                             orderBuffer=lists[1].handle)
    device.synchronize()
    offsets, order, _ = R.group_rows(ids, E)
    h = expected(a[order // fan], w1, offsets, fill=0)
    want = expected(h, w2, offsets, order, fill=0)
    assert R.same_bits(hb.get(np.float16).reshape(rows, F), h)
    assert R.same_bits(cb.get(np.float16).reshape(rows, K), want)


# ------------------------------------------------------------------------------------------ in use

def test_calls_in_a_row_do_not_disturb_each_other():
    """Sizes up and down on one context, nothing waited for in between: scratch is shared and reused."""
    jobs = []
    for i, (M, K, N) in enumerate([(300, 1000, 500), (1, 4096, 600), (33, 130, 90), (2, 700, 3000), (300, 1000, 500), (17, 9000, 64)]):
        a, w = data(i, M, K, N, np.float32)
        jobs.append((a, w, pack(w), DevBuf.of(a), DevBuf(M * N * 4)))
    for _ in range(3):
        for a, w, packed, ab, cb in jobs:
            device.int8Matmul(device.DTYPE_F32, ab.handle, packed.handle, cb.handle, a.shape[0], w.shape[1], a.shape[1])
    device.synchronize()
    for a, w, packed, ab, cb in jobs:
        assert R.same_bits(cb.get(np.float32).reshape(a.shape[0], w.shape[1]), R.product(a, w))


def test_captured_graphs_share_scratch_and_outlive_its_growth():
    """Two graphs replayed in turn on new inputs, then again after a larger call has taken more scratch."""
    E, K, N, T, fan = 5, 300, 200, 50, 2
    rows = T * fan
    a, w = data(0, T, K, N, np.float32, experts=E)
    packed = pack(w)
    a1, w1 = data(1, 9, 2000, 300, np.float32)
    packed1 = pack(w1)
    ab, ib, ab1 = DevBuf.of(a), DevBuf(rows * 4), DevBuf.of(a1)
    lists = [DevBuf((E + 1) * 4), DevBuf(rows * 4), DevBuf(rows * 4)]
    cb, cb1 = DevBuf.of(np.zeros((rows, N), np.float32)), DevBuf.of(np.zeros((9, 300), np.float32))

    def one():
        device.groupRows(ib.handle, *(x.handle for x in lists), rows, E)
        device.int8MatmulGrouped(device.DTYPE_F32, ab.handle, packed.handle, lists[0].handle, cb.handle, rows, N, K, E,
                                 positionBuffer=lists[2].handle, orderBuffer=lists[1].handle, fan=fan)

    def two():
        device.int8Matmul(device.DTYPE_F32, ab1.handle, packed1.handle, cb1.handle, 9, 300, 2000)

    graphs = []
    for job in (one, two):
        device.upload(ib.handle, np.zeros(rows, np.int32))
        job()
        device.synchronize()
        device.graphBegin()
        job()
        graphs.append(device.graphEnd())
    rng = np.random.default_rng(3)

    def check():
        ids = rng.integers(-1, E, (T, fan)).astype(np.int32)
        x, x1 = rng.standard_normal((T, K)).astype(np.float32), rng.standard_normal((9, 2000)).astype(np.float32)
        for b, v in ((ib, ids), (ab, x), (ab1, x1), (cb, np.zeros((rows, N), np.float32))):
            device.upload(b.handle, v)
        device.graphLaunch(graphs[0])
        device.graphLaunch(graphs[1])
        device.graphLaunch(graphs[0])
        device.synchronize()
        assert device.kernelStatus() == 0
        offsets, order, _ = R.group_rows(ids, E)
        assert R.same_bits(cb.get(np.float32).reshape(rows, N), expected(x[order // fan], w, offsets, order, fill=0))
        assert R.same_bits(cb1.get(np.float32).reshape(9, 300), R.product(x1, w1))

    check()
    check()
    big, wbig = data(8, 3000, 4000, 64, np.float32)
    want = R.product(big, wbig)
    assert R.same_bits(matmul(big, pack(wbig), 64), want)
    check()
    assert R.same_bits(matmul(big, pack(wbig), 64), want)
    for g in graphs:
        device.graphDestroy(g)


def test_two_contexts_at_once():
    """A second context has a stream and scratch of its own: its calls may run beside the first one's."""
    import ctypes as C
    import torch
    lib = device.lib
    other = lib.smith_init_device(device.deviceIndex())
    assert other
    a, w = data(21, 65, 3000, 500, np.float32)
    want, packed = R.product(a, w), pack(w)
    first = DevBuf.of(a), DevBuf(65 * 500 * 4)
    x = torch.from_numpy(a).cuda()
    y = torch.zeros(65, 500, device="cuda")
    torch.cuda.synchronize()
    handles = [lib.smith_wrap_device_memory(other, C.c_void_p(p), n) for p, n in
               ((x.data_ptr(), a.nbytes), (device.devicePtr(packed.handle), packed.nbytes), (y.data_ptr(), 65 * 500 * 4))]
    for _ in range(20):
        device.int8Matmul(device.DTYPE_F32, first[0].handle, packed.handle, first[1].handle, 65, 500, 3000)
        assert lib.smith_int8_matmul(other, 0, handles[0], handles[1], handles[2], 65, 500, 3000, 0, 0) == 0
    device.synchronize()
    assert lib.smith_synchronize(other) == 0
    assert R.same_bits(first[1].get(np.float32).reshape(65, 500), want)
    assert R.same_bits(y.cpu().numpy(), want)
    for h in handles:
        lib.smith_release_buffer(h)
    lib.smith_destroy(other)


def test_same_call_gives_the_same_bits_every_time():
    """Shared tiles are joined by whichever worker is last: whole numbers, so it does not show."""
    for M, K, N in [(1, 4096, 1024), (24, 9000, 384), (300, 7000, 700)]:
        a, w = data(M, M, K, N, np.float16)
        packed, want = pack(w), R.product(a, w)
        for _ in range(25):
            assert R.same_bits(matmul(a, packed, N), want)


def test_capture_of_a_call_that_needs_more_scratch_is_refused():
    """More rows than any other test: the scratch has to grow, which a capture cannot do."""
    M, K, N = 100_000, 640, 8
    a, w = data(0, M, K, N, np.float16)
    packed, ab, cb = pack(w), DevBuf.of(a), DevBuf(M * N * 2)
    device.graphBegin()
    try:
        with pytest.raises(device.SmithError, match="before graph capture"):
            device.int8Matmul(device.DTYPE_F16, ab.handle, packed.handle, cb.handle, M, N, K)
    finally:
        device.graphDestroy(device.graphEnd())
    device.int8Matmul(device.DTYPE_F16, ab.handle, packed.handle, cb.handle, M, N, K)
    device.synchronize()
    assert R.same_bits(cb.get(np.float16).reshape(M, N), R.product(a, w))


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_operators_on_tensors(dtype):
    np_dtype = np.float16 if dtype == "f16" else np.float32

    def tensor(x):
        t = smith.create(list(x.shape), dtype)
        t.data[:] = x.reshape(-1).view(np.uint16) if dtype == "f16" else x.reshape(-1)
        return t

    def values(t):
        v = smith.toNumpy(t)
        return v.view(np.float16) if dtype == "f16" else v

    for M, K, N in [(1, 256, 300), (50, 130, 70), (0, 64, 64)]:
        a, w = data(M, M, K, N, np_dtype)
        rec = smith.quantizeInt8(tensor(w))
        assert (rec.K, rec.N, rec.experts) == (K, N, 1)
        assert R.same_bits(values(smith.matmulInt8(tensor(a), rec)), R.product(a, w).reshape(M, N))
        device.releaseBuffer(rec.buffer)
    E, T, fan, K, N = 4, 20, 2, 100, 90
    a, w = data(9, T, K, N, np_dtype, experts=E)
    rec = smith.quantizeInt8(tensor(w))
    ids = np.random.default_rng(0).integers(-1, E, (T, fan)).astype(np.int32)
    offsets, order, position = R.group_rows(ids, E)
    groups = smith.groupRows(smith.tensorFrom(ids, [T, fan], "i32"), E)
    for name, want in (("offsets", offsets), ("order", order), ("position", position)):
        assert np.array_equal(smith.toNumpy(groups[name]), want)
    got = values(smith.matmulInt8Grouped(tensor(a), rec, groups))
    a_sorted = np.ascontiguousarray(a[order // fan])
    assert R.same_bits(got, expected(a_sorted, w, offsets, fill=0))
    got = values(smith.matmulInt8Grouped(tensor(a_sorted), rec, groups, gather=False, scatter=True))
    assert R.same_bits(got, expected(a_sorted, w, offsets, order, fill=0))
    with pytest.raises(ValueError, match="matmulInt8Grouped"):
        smith.matmulInt8(tensor(a), rec)


def test_profiled_operators_report_their_kernels():
    a, w = data(1, 8, 256, 128, np.float32)
    rec = smith.quantizeInt8(smith.tensorFrom(w, [256, 128]))
    res = smith.profileFn(lambda: smith.matmulInt8(smith.tensorFrom(a, [8, 256]), rec))
    (entry,) = [k for k in res["kernels"] if k["kernel"] == "matmul_int8"]
    assert entry["calls"] == 1 and entry["tflops"] >= 0 and entry["gbs"] > 0


def test_profiling_takes_empty_batches():
    """No rows: nothing is launched, and the timed submit reports it like any other."""
    rec = smith.quantizeInt8(smith.tensorFrom(np.ones((64, 32), np.float32), [64, 32]))
    ids = smith.create([0], "i32")

    def calls():
        groups = smith.groupRows(ids, 1)
        return smith.matmulInt8(smith.create([0, 64]), rec), smith.matmulInt8Grouped(smith.create([0, 64]), rec, groups), groups

    res = smith.profileFn(calls)
    one, two, groups = res["result"]
    assert one.shape == [0, 32] and two.shape == [0, 32] and smith.toNumpy(groups.offsets).tolist() == [0, 0]
    assert {k["kernel"] for k in res["kernels"]} == {"matmul_int8", "matmul_int8_grouped", "group_rows"}


def test_packed_weights_on_disk(tmp_path):
    a, w = data(3, 6, 130, 200, np.float32, experts=None)
    rec = smith.quantizeInt8(smith.tensorFrom(w, [130, 200]))
    q8 = smith.quantizeQ8(smith.tensorFrom(w, [130, 200]))
    path = str(tmp_path / "weights")
    smith.saveQuantized({"a": ("i8", rec), "b": ("q8", q8)}, path)
    back = smith.loadQuantized(path)
    kind, again = back["a"]
    assert kind == "i8" and back["b"][0] == "q8"
    assert np.array_equal(device.download(again.buffer, again.totalBytes), device.download(rec.buffer, rec.totalBytes))
    got = smith.toNumpy(smith.matmulInt8(smith.tensorFrom(a, [6, 130]), again))
    assert R.same_bits(got, R.product(a, w))


def test_refusals():
    """Each wrong call names its fault and launches nothing."""
    M, K, N, E = 8, 64, 32, 2
    a, w = data(0, M, K, N, np.float32, experts=E)
    packed, ab, cb = pack(w), DevBuf.of(a), DevBuf(M * N * 4)
    ob, lb, ids = DevBuf.of(np.array([0, 4, 8], np.int32)), DevBuf.of(np.arange(M, dtype=np.int32)), DevBuf.of(np.zeros(M, np.int32))
    f32 = device.DTYPE_F32
    before = device.launchCount()

    def refused(text, fn, *args, **kw):
        with pytest.raises(device.SmithError, match=text):
            fn(*args, **kw)

    mm, gm = device.int8Matmul, device.int8MatmulGrouped
    refused("dtype", mm, 2, ab.handle, packed.handle, cb.handle, M, N, K)
    refused("K = 0", mm, f32, ab.handle, packed.handle, cb.handle, M, N, 0)
    refused("K = 131073", mm, f32, ab.handle, packed.handle, cb.handle, M, N, 131073)
    refused("N = 0", mm, f32, ab.handle, packed.handle, cb.handle, M, 0, K)
    refused("A holds", mm, f32, ab.handle, packed.handle, cb.handle, M + 1, N, K)
    refused("C holds", mm, f32, ab.handle, packed.handle, cb.handle, M, N + 1, K)
    refused("pitches", mm, f32, ab.handle, packed.handle, cb.handle, M, N, K, K - 1)
    refused("pitches", mm, f32, ab.handle, packed.handle, cb.handle, M, N, K, 0, N - 1)
    refused("pitches", mm, f32, ab.handle, packed.handle, cb.handle, M, N, K, 1 << 40)
    refused("rows", mm, f32, ab.handle, packed.handle, cb.handle, 1 << 31, N, K)
    refused("packed weights hold", gm, f32, ab.handle, cb.handle, ob.handle, cb.handle, M, N, K, E)
    refused("overlaps", gm, f32, ab.handle, packed.handle, ob.handle, packed.handle, M, N, K, E)
    small = device.wrapDeviceMemory(device.devicePtr(ob.handle), 8)
    refused("offsets holds", gm, f32, ab.handle, packed.handle, small, cb.handle, M, N, K, E)
    refused("offsets are missing", gm, f32, ab.handle, packed.handle, None, cb.handle, M, N, K, E)
    refused("experts", gm, f32, ab.handle, packed.handle, ob.handle, cb.handle, M, N, K, 1025)
    refused("fan", gm, f32, ab.handle, packed.handle, ob.handle, cb.handle, M, N, K, E, fan=2)
    refused("fan", gm, f32, ab.handle, packed.handle, ob.handle, cb.handle, M, N, K, E, positionBuffer=lb.handle, fan=3)
    refused("fan", gm, f32, ab.handle, packed.handle, ob.handle, cb.handle, M, N, K, E, positionBuffer=lb.handle, fan=0)
    refused("position holds", gm, f32, ab.handle, packed.handle, ob.handle, cb.handle, M, N, K, E, positionBuffer=ob.handle)
    refused("order holds", gm, f32, ab.handle, packed.handle, ob.handle, cb.handle, M, N, K, E, orderBuffer=ob.handle)
    odd = device.wrapDeviceMemory(device.devicePtr(cb.handle) + 2, M * N * 4 - 2)
    refused("aligned", mm, f32, ab.handle, packed.handle, odd, M - 1, N, K)
    off = device.wrapDeviceMemory(device.devicePtr(packed.handle) + 8, packed.nbytes - 8)
    refused("16 bytes", mm, f32, ab.handle, off, cb.handle, M, N, K)
    shared = device.alloc(M * K * 4)
    refused("device side", mm, f32, shared, packed.handle, cb.handle, M, N, K)
    refused("needs", device.int8Pack, f32, ab.handle, packed.handle, K * 1000, N, E)
    refused("overlap", device.int8Pack, f32, packed.handle, packed.handle, 8, 8, 1)
    refused("experts", device.int8PackedBytes, K, N, 0)
    refused("experts", device.groupRows, ids.handle, ob.handle, lb.handle, lb.handle, M, 0)
    refused("experts", device.groupRows, ids.handle, ob.handle, lb.handle, lb.handle, M, 1025)
    refused("overlap", device.groupRows, ids.handle, ob.handle, lb.handle, lb.handle, M, E)
    refused("overlaps the ids", device.groupRows, ids.handle, ob.handle, ids.handle, lb.handle, M, E)
    refused("buffer 0 holds", device.groupRows, ob.handle, ob.handle, ids.handle, lb.handle, M, E)
    for h in (small, odd, off, shared):
        device.releaseBuffer(h)
    assert device.launchCount() == before


def test_no_rows_is_no_launch():
    packed, b = pack(np.ones((8, 8), np.float32)), DevBuf(64)
    before = device.launchCount()
    device.int8Matmul(device.DTYPE_F32, b.handle, packed.handle, b.handle, 0, 8, 8)
    assert device.launchCount() == before

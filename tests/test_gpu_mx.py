"""Microscaled rows and weights on the GPU against a plain statement of the format in float64 (``mx_util``).

Tolerances.  Quantisation and reading back have one right answer: codes and scales are compared bit by bit.  A product's
operands are the numbers that the codes stand for, so nothing is left but float32 sums: every product of two elements is exact
in the tensor core and an output is a sum of K of them, taken 32 or more at a time, so its error is at most (K / 32 + 8)
roundings of 2^-22 (two bits are granted to the tensor core's way of adding) times the sum of the terms' magnitudes.  Rows that
come out in the format may lie ``mx_util.rounding`` from the float64 ones, plus that error."""
import numpy as np
import pytest
import torch

import mx_util

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from tinyinfer_b200.kernels import cuda_ops
    return cuda_ops("cuda:0")


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def activations(seed, rows, k, dtype=torch.float32):
    g = gen(seed)
    x = torch.randn(rows, k, device="cuda", generator=g)
    x = x * torch.exp(torch.randn(k, device="cuda", generator=g)) * torch.exp(2 * torch.randn(rows, 1, device="cuda", generator=g))
    return x.to(dtype)


def same_format(q, x):
    """``q`` holds exactly the plain quantisation of ``x``, zeros behind its columns included."""
    codes, scales = mx_util.unpack(q)
    want_codes, want_scales = mx_util.quantize(x.double().cpu().numpy(), q.bits)
    finite = np.repeat(want_scales != 255, 32, axis=1)
    np.testing.assert_array_equal(scales, want_scales)
    np.testing.assert_array_equal(codes[finite], want_codes[finite])


def fine(ops):
    torch.cuda.synchronize()
    ops.check_status()


# ---- quantisation --------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("rows, k, skip, wide", [(1, 1, 0, 0), (1, 31, 0, 0), (1, 32, 0, 0), (3, 33, 0, 0), (5, 128, 0, 0),
                                                 (129, 200, 0, 0), (257, 1000, 0, 0), (2, 4096, 0, 0), (33, 260, 1, 0),
                                                 (33, 260, 8, 0), (33, 260, 8, 4), (17, 255, 3, 2), (300, 136, 16, 8)])
def test_quantize(ops, dtype, bits, rows, k, skip, wide):
    x = activations(rows + k, rows, skip + k + wide, dtype)[:, skip:skip + k]
    q = ops.mx_quantize(x, bits)
    assert q.bits == bits and q.cols == k and q.rows == rows
    same_format(q, x)
    fine(ops)


@pytest.mark.parametrize("shift", [0, 1])                      # rows on 16 bytes and off them
@pytest.mark.parametrize("bits", [4, 8])
def test_quantize_extremes(ops, bits, shift):
    x = torch.zeros(12, 128 + shift, device="cuda")
    x = x[:, shift:]
    x[1] = 1e-45                                               # below float32's normal range
    x[2] = 3e-39 * torch.arange(128, device="cuda")
    x[3] = 3.3e38
    x[4] = torch.linspace(-8, 8, 128, device="cuda")           # ties of both element types among them
    x[5] = torch.arange(128, device="cuda") * 0.25 - 16
    x[6, 0] = float("inf")
    x[7, 40] = float("nan")
    x[8, 127] = -float("inf")
    x[9, :32] = -0.0
    x[10] = torch.finfo(torch.float32).min
    x[11] = 2.0 ** torch.arange(-64, 64, device="cuda")
    q = ops.mx_quantize(x, bits)
    same_format(q, x)
    got = ops.mx_dequantize(q, torch.float32).double().cpu().numpy()
    np.testing.assert_array_equal(got, mx_util.values_of(q))   # NaN in the blocks that hold an infinity or NaN, and there alone
    assert np.isnan(got[6, :32]).all() and not np.isnan(got[6, 32:]).any()
    fine(ops)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("rows, k", [(1, 1), (5, 33), (130, 264), (64, 1000)])
def test_every_code_reads_back(ops, dtype, bits, rows, k):
    rng = np.random.RandomState(rows)
    codes = rng.randint(0, 1 << bits, (rows, mx_util.padded(k)))
    if bits == 8:
        codes[codes % 128 == 127] = 0                          # the element type's own NaN
    scales = rng.randint(100, 140, (rows, mx_util.padded(k) // 32))
    from tinyinfer_b200.kernels import MxRows
    held, tiles = mx_util.pack(codes, scales, bits)
    q = MxRows(held.cuda(), tiles.cuda(), bits, k)
    guard = torch.full((rows, k + 6), 7.0, device="cuda", dtype=dtype)
    out = ops.mx_dequantize(q, out=guard[:, 3:3 + k])
    np.testing.assert_array_equal(out.double().cpu().numpy(), mx_util.numbers(codes, scales, bits)[:, :k])
    assert (guard[:, :3] == 7).all() and (guard[:, 3 + k:] == 7).all()
    np.testing.assert_array_equal(ops.mx_dequantize(q, dtype).double().cpu().numpy(), out.double().cpu().numpy())


def test_quantize_rows_far_apart(ops):
    step = (1 << 30) + 8                                       # the third row starts behind 2^31 elements
    room = torch.empty(2 * step + 256, dtype=torch.bfloat16, device="cuda")
    x = room.as_strided((3, 200), (step, 1))
    x.copy_(activations(5, 3, 200, torch.bfloat16))
    same_format(ops.mx_quantize(x, 8), x)


@pytest.mark.parametrize("bits", [4, 8])
def test_outputs_stay_inside(ops, bits):
    from tinyinfer_b200.kernels import MxRows
    rows, k = 5, 200
    room_c = torch.full((rows + 2, 256 * bits // 8), 0xAB, dtype=torch.uint8, device="cuda")
    room_s = torch.full((3, 2, 512), 0xAB, dtype=torch.uint8, device="cuda")
    q = MxRows(room_c[1:1 + rows], room_s[1:2], bits, k)
    x = activations(1, rows, k)
    assert ops.mx_quantize(x, bits, out=q) is q
    same_format(q, x)
    ops.mx_rmsnorm(x, torch.ones(k, device="cuda"), 1e-6, bits, out=q)
    w = ops.mx_pack_gate_up(torch.randn(k, 100, device="cuda"), torch.randn(k, 100, device="cuda"))
    ops.mx_linear_glu(ops.mx_quantize(activations(2, rows, 100), 8), w, k, bits, out=q)
    fine(ops)
    for room in (room_c, room_s):
        assert (room[0] == 0xAB).all() and (room[-1] == 0xAB).all()


# ---- the norm ------------------------------------------------------------------------------------
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("delta", [None, torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows, k, skip", [(1, 1, 0), (3, 31, 0), (2, 128, 0), (7, 333, 0), (130, 1024, 0), (5, 4096, 0),
                                           (3, 8200, 0), (2, 32768, 0), (9, 500, 4), (9, 501, 3)])
def test_rmsnorm(ops, bits, delta, rows, k, skip):
    room = activations(k, rows, skip + k)
    x = room[:, skip:]
    weight = 1 + 0.5 * torch.randn(k, device="cuda", generator=gen(3))
    d = None if delta is None else activations(k + 1, rows, skip + k, delta)[:, skip:]
    want_x = x.clone() if d is None else x + d.float()
    before = room[:, :skip].clone()
    q = ops.mx_rmsnorm(x, weight, 1e-5, bits, delta=d)
    fine(ops)
    assert torch.equal(x, want_x) and torch.equal(room[:, :skip], before)
    y = want_x.double().cpu().numpy()
    exact = y / np.sqrt((y * y).mean(axis=1, keepdims=True) + 1e-5) * weight.double().cpu().numpy()
    off = np.abs(mx_util.values_of(q) - exact)
    assert (off <= mx_util.rounding(exact, bits) + 1e-5 * np.abs(exact)).all()
    codes, _ = mx_util.unpack(q)
    assert not codes[:, k:].any()


def test_rmsnorm_of_zeros_and_infinities(ops):
    x = torch.zeros(3, 160, device="cuda")
    x[1, 5], x[2, 7] = float("inf"), float("nan")
    got = ops.mx_dequantize(ops.mx_rmsnorm(x, torch.ones(160, device="cuda"), 1e-6))
    assert (got[0] == 0).all() and got[1, 5].isnan() and got[2].isnan().all()


# ---- products ------------------------------------------------------------------------------------
def bound(a, w, k):
    """The products' tolerance, element by element."""
    return (k / 32 + 8) * 2.0 ** -22 * (np.abs(a) @ np.abs(w).T)


SIZES = [(1, 1, 1), (1, 128, 128), (1, 129, 4096), (2, 64, 31), (7, 200, 300), (16, 520, 1000), (17, 127, 256), (33, 130, 129),
         (64, 256, 640), (65, 300, 384), (100, 520, 1152), (128, 128, 2048), (129, 260, 200), (200, 640, 1100), (256, 512, 512),
         (257, 256, 128), (300, 200, 100), (511, 513, 900), (513, 1100, 260), (1000, 300, 2000)]


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("m, n, k", SIZES)
def test_linear(ops, bits, m, n, k):
    a, w = ops.mx_quantize(activations(m, m, k), bits), ops.mx_pack_linear(torch.randn(n, k, device="cuda", generator=gen(n)))
    av, wv = mx_util.values_of(a), mx_util.values_of(w)
    exact, tol = av @ wv.T, bound(av, wv, k)
    room = torch.full((m, n + 5), 3.0, device="cuda")
    for add in (False, True):
        for out in (torch.randn(m, n, device="cuda", generator=gen(7)), room[:, 2:2 + n]):
            old = out.double().cpu().numpy()
            got = ops.mx_linear(a, w, out, accumulate=add)
            fine(ops)
            want = exact + old if add else exact
            off = np.abs(got.double().cpu().numpy() - want)
            assert (off <= tol + 2.0 ** -23 * np.abs(want)).all(), off.max()
    assert (room[:, :2] == 3).all() and (room[:, 2 + n:] == 3).all()


# enough tiles of 256 x 256 for pairs of SMs, none of them whole in every direction
MANY = [(1100, 2117, 300), (2600, 1001, 129), (700, 4000, 1100), (300, 5121, 256), (129, 10400, 40)]


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("m, n, k", MANY)
def test_linear_of_many_tiles(ops, bits, m, n, k):
    a, w = ops.mx_quantize(activations(m, m, k), bits), ops.mx_pack_linear(torch.randn(n, k, device="cuda", generator=gen(n)))
    av, wv = mx_util.values_of(a), mx_util.values_of(w)
    exact, tol = av @ wv.T, bound(av, wv, k)
    room = torch.full((m + 2, n + 5), 3.0, device="cuda")
    out = room[1:1 + m, 2:2 + n]
    for add in (False, True):
        old = out.double().cpu().numpy()
        ops.mx_linear(a, w, out, accumulate=add)
        fine(ops)
        want = exact + old if add else exact
        assert (np.abs(out.double().cpu().numpy() - want) <= tol + 2.0 ** -23 * np.abs(want)).all()
    first = out.clone()
    ops.mx_linear(a, w, out)
    assert torch.equal(ops.mx_linear(a, w, out, accumulate=True), first)             # the same bits again
    assert (room[[0, -1]] == 3).all() and (room[:, :2] == 3).all() and (room[:, 2 + n:] == 3).all()


# Every number of parts of K and of blocks of an SM: tiles of 128 weight rows by stages of K (128 elements beside rows of 8
# bits, 256 beside 4): 297 x 2, 223 x 8, 223 x 8, 149 x 25, 67 x 64, 35 x 16, 76 x 21, 32 x 48, 3 x 65, 35 x 16, 17 x 12, 9 x 9
SPLITS = [(5, 38001, 160, 8), (8, 28500, 900, 8), (20, 28500, 900, 8), (3, 18990, 3081, 8), (9, 8500, 8103, 8), (31, 4400, 2000, 8),
          (16, 9700, 2600, 8), (7, 4000, 6050, 8), (32, 300, 8203, 8), (8, 4401, 4000, 4), (1, 2100, 1500, 8), (2, 1100, 1100, 8),
          (50, 4000, 6050, 8), (4, 38001, 300, 4)]


@pytest.mark.parametrize("m, n, k, bits", SPLITS)
def test_linear_of_every_split(ops, m, n, k, bits):
    a, w = ops.mx_quantize(activations(m, m, k), bits), ops.mx_pack_linear(torch.randn(n, k, device="cuda", generator=gen(n)))
    av, wv = mx_util.values_of(a), mx_util.values_of(w)
    exact, tol = av @ wv.T, bound(av, wv, k)
    room = torch.full((m + 2, n + 5), 3.0, device="cuda")
    out = room[1:1 + m, 2:2 + n]
    ops.mx_linear(a, w, out)
    first = out.clone()
    for add in (False, True):
        want = exact + out.double().cpu().numpy() if add else exact
        ops.mx_linear(a, w, out, accumulate=add)
        fine(ops)
        assert (np.abs(out.double().cpu().numpy() - want) <= tol + 2.0 ** -23 * np.abs(want)).all()
        assert add or torch.equal(out, first)                                        # the same bits again
    assert (room[[0, -1]] == 3).all() and (room[:, :2] == 3).all() and (room[:, 2 + n:] == 3).all()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("m, n", [(1100, 2117), (300, 200)])
def test_products_of_many_rows_keep_nan_in_its_row_and_column(ops, bits, m, n):
    x, w = activations(1, m, 300), torch.randn(n, 300, device="cuda", generator=gen(2))
    x[m - 1, 290] = float("nan")
    w[150, 3] = float("inf")
    a = ops.mx_quantize(x, bits)
    bad = ops.mx_linear(a, ops.mx_pack_linear(w), torch.empty(m, n, device="cuda")).isnan()
    assert bad[m - 1].all() and bad[:, 150].all() and bad.sum() == n + m - 1
    # gated rows: a NaN takes its block of 32 columns along, and in the row of NaN all of them
    q = ops.mx_dequantize(ops.mx_linear_glu(a, ops.mx_pack_gate_up(w, torch.ones_like(w)), n))
    fine(ops)
    bad = q.isnan()
    assert bad[m - 1].all() and bad[:, 128:160].all() and bad.sum() == n + 32 * (m - 1)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("m", [3, 40, 300])
def test_linear_keeps_nan_in_its_row_and_column(ops, bits, m):
    x, w = activations(1, m, 300), torch.randn(200, 300, device="cuda", generator=gen(2))
    x[m - 1, 290] = float("inf")
    w[150, 3] = float("nan")
    out = ops.mx_linear(ops.mx_quantize(x, bits), ops.mx_pack_linear(w), torch.empty(m, 200, device="cuda"))
    fine(ops)
    bad = out.isnan()
    assert bad[m - 1].all() and bad[:, 150].all() and bad.sum() == 200 + m - 1


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("m, n, k", [(5, 400, 3000), (64, 300, 4096), (300, 300, 700)])
def test_linear_gives_the_same_bits_again(ops, bits, m, n, k):
    a, w = ops.mx_quantize(activations(m, m, k), bits), ops.mx_pack_linear(torch.randn(n, k, device="cuda", generator=gen(n)))
    first = ops.mx_linear(a, w, torch.empty(m, n, device="cuda"))
    for _ in range(20):
        assert torch.equal(ops.mx_linear(a, w, torch.empty(m, n, device="cuda")), first)
    fine(ops)


def test_linear_large_scales(ops):
    """Blocks of very different sizes side by side: what is far below the rest of a sum vanishes, nothing overflows early."""
    x = torch.randn(20, 512, device="cuda", generator=gen(1)) * 2.0 ** torch.linspace(-60, 60, 512, device="cuda")
    w = torch.randn(130, 512, device="cuda", generator=gen(2)) * 2.0 ** torch.linspace(60, -60, 512, device="cuda")
    a, b = ops.mx_quantize(x, 8), ops.mx_pack_linear(w)
    got = ops.mx_linear(a, b, torch.empty(20, 130, device="cuda")).double().cpu().numpy()
    av, bv = mx_util.values_of(a), mx_util.values_of(b)
    assert (np.abs(got - av @ bv.T) <= bound(av, bv, 512)).all()


def test_linear_rows_far_apart(ops):
    step = (1 << 29) + 4                                       # the fifth row of out starts behind 2^31 floats
    room = torch.empty(4 * step + 200, device="cuda")
    out = room.as_strided((5, 150), (step, 1))
    a, w = ops.mx_quantize(activations(1, 5, 256), 8), ops.mx_pack_linear(torch.randn(150, 256, device="cuda", generator=gen(3)))
    want = ops.mx_linear(a, w, torch.empty(5, 150, device="cuda"))
    assert torch.equal(ops.mx_linear(a, w, out), want)


def glu_exact(a, gate, up):
    g, u = a @ gate.T, a @ up.T
    with np.errstate(over="ignore"):
        return g / (1 + np.exp(-g)) * u, g, u


@pytest.mark.parametrize("obits", [4, 8])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("m, n, k", [(1, 1, 1), (1, 128, 128), (5, 100, 300), (16, 200, 1000), (33, 65, 256), (64, 384, 640),
                                     (100, 130, 129), (129, 257, 512), (256, 128, 200), (300, 300, 384), (700, 500, 100)])
def test_glu(ops, obits, bits, m, n, k):
    gate = torch.randn(n, k, device="cuda", generator=gen(n)) * k ** -0.5
    up = torch.randn(n, k, device="cuda", generator=gen(n + 1)) * k ** -0.5
    a, w = ops.mx_quantize(activations(m, m, k), bits), ops.mx_pack_gate_up(gate, up)
    q = ops.mx_linear_glu(a, w, n, obits)
    fine(ops)
    assert q.bits == obits and q.cols == n and q.rows == m
    av = mx_util.values_of(a)
    gv, uv = (mx_util.values_of(ops.mx_quantize(t, 4)) for t in (gate, up))
    exact, g, u = glu_exact(av, gv, uv)
    # an error e of the gate changes silu by at most 1.1 e, one of up is multiplied by silu <= |gate|; 1e-5 for the
    # approximate exponential and reciprocal
    off_by = 1.1 * bound(av, gv, k) * np.abs(u) + np.abs(g) * bound(av, uv, k) + 1e-5 * np.abs(exact)
    off = np.abs(mx_util.values_of(q) - exact)
    assert (off <= mx_util.rounding(np.abs(exact) + off_by, obits) + off_by).all()
    codes, scales = mx_util.unpack(q)
    assert not codes[:, n:].any() and (scales != 255).all()


# tiles by stages 149 x 16, 297 x 2, 35 x 16, 80 x 21, 17 x 8, 6 x 50, 17 x 4
@pytest.mark.parametrize("m, n, k", [(3, 9520, 2000), (8, 18960, 200), (10, 2200, 2000), (30, 5100, 2600), (6, 1030, 1000),
                                     (9, 380, 6300), (60, 1030, 500)])
def test_glu_of_every_split(ops, m, n, k):
    test_glu(ops, 8, 8, m, n, k)


@pytest.mark.parametrize("m", [3, 300])
def test_glu_of_large_gates(ops, m):
    """silu at both ends: zero for very negative gates and the gate itself for large ones; NaN only where an input is."""
    x = torch.ones(m, 32, device="cuda")
    gate = torch.full((64, 32), -1000.0, device="cuda")
    gate[32:] = 1000.0
    up = torch.ones(64, 32, device="cuda")
    w = ops.mx_pack_gate_up(gate, up)
    got = ops.mx_dequantize(ops.mx_linear_glu(ops.mx_quantize(x, 8), w, 64, 8)).float()
    assert (got[:, :32] == 0).all()
    # 1000 saturates to 6 * 128 in 4 bits; (32 * 768) * 32 has three significant bits
    assert (got[:, 32:] == 768 * 32 * 32).all()
    x[m - 1, 3] = float("nan")
    got = ops.mx_dequantize(ops.mx_linear_glu(ops.mx_quantize(x, 8), w, 64, 8))
    fine(ops)
    assert got[m - 1].isnan().all() and not got[:m - 1].isnan().any()


# ---- streams, graphs, empty inputs, refusals -----------------------------------------------------
def test_on_a_stream_of_its_own_and_in_a_graph(ops):
    x, weight = activations(1, 40, 512), torch.ones(512, device="cuda")
    delta = activations(2, 40, 512, torch.bfloat16)
    gate_up = ops.mx_pack_gate_up(torch.randn(384, 512, device="cuda") * 0.05, torch.randn(384, 512, device="cuda") * 0.05)
    down = ops.mx_pack_linear(torch.randn(512, 384, device="cuda") * 0.05)

    def layer(x):
        h = ops.mx_rmsnorm(x, weight, 1e-6, 8, delta=delta)
        ops.mx_linear(ops.mx_linear_glu(h, gate_up, 384), down, x, accumulate=True)
        return x

    want = layer(x.clone())
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        mine = x.clone()
        stream.synchronize()
        got = layer(mine)
    stream.synchronize()
    assert torch.equal(got, want)
    held, graph = x.clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer(held)
    for _ in range(3):
        held.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, want)
    fine(ops)


def test_one_row_for_all(ops):
    """Rows that share their memory may be read: a delta that is one row, an input that is."""
    x, one = activations(1, 6, 160), activations(2, 1, 160)
    y = x.clone()
    got = ops.mx_dequantize(ops.mx_rmsnorm(x, torch.ones(160, device="cuda"), 1e-6, delta=one.expand(6, 160)))
    want = ops.mx_dequantize(ops.mx_rmsnorm(y, torch.ones(160, device="cuda"), 1e-6, delta=one.repeat(6, 1)))
    assert torch.equal(got, want) and torch.equal(x, y)
    same_format(ops.mx_quantize(one.expand(6, 160), 4), one.repeat(6, 1))


def test_held_back_products_run_first(ops):
    """A product that another part let the kernel set hold back is in the residual before the norm reads it."""
    from tinyinfer_b200.kernels import CudaOps
    mine = CudaOps("cuda:0")
    a, w = (torch.randn(s, device="cuda", generator=gen(i)).bfloat16() for i, s in enumerate(((4, 256), (512, 256))))
    x, ones = torch.randn(4, 512, device="cuda", generator=gen(5)), torch.ones(512, device="cuda")
    want = x.clone()
    mine.linear(a, w, want, accumulate=True)
    want = mine.mx_dequantize(mine.mx_rmsnorm(want, ones, 1e-6))
    mine.linear(a, w, x, accumulate=True, may_defer=True)
    assert mine._pending is not None
    assert torch.equal(mine.mx_dequantize(mine.mx_rmsnorm(x, ones, 1e-6)), want)
    assert mine._pending is None


def test_no_rows(ops):
    w = ops.mx_pack_linear(torch.randn(8, 64, device="cuda"))
    q = ops.mx_quantize(torch.empty(0, 64, device="cuda"), 8)
    assert q.rows == 0 and ops.mx_dequantize(q).shape == (0, 64)
    assert ops.mx_linear(q, w, torch.empty(0, 8, device="cuda")).shape == (0, 8)
    assert ops.mx_linear_glu(q, ops.mx_pack_gate_up(*torch.randn(2, 8, 64, device="cuda")), 8).rows == 0
    assert ops.mx_rmsnorm(torch.empty(0, 64, device="cuda"), torch.ones(64, device="cuda"), 1e-6).rows == 0
    fine(ops)


def test_refusals(ops):
    from tinyinfer_b200.kernels import KernelError, MxRows
    x = torch.randn(4, 64, device="cuda")
    a, w = ops.mx_quantize(x, 8), ops.mx_pack_linear(torch.randn(8, 64, device="cuda"))
    out, ones = torch.empty(4, 8, device="cuda"), torch.ones(64, device="cuda")
    glu = ops.mx_pack_gate_up(*torch.randn(2, 8, 64, device="cuda"))
    calls = [
        lambda: ops.mx_quantize(x, 5), lambda: ops.mx_quantize(x.half(), 8), lambda: ops.mx_quantize(x.cpu(), 8),
        lambda: ops.mx_quantize(x[0], 8), lambda: ops.mx_quantize(x.T, 8), lambda: ops.mx_quantize(x[:, :0], 8),
        lambda: ops.mx_quantize(x, 4, out=a), lambda: ops.mx_quantize(x[:3], 8, out=a), lambda: ops.mx_quantize("x", 8),
        lambda: ops.mx_dequantize(a, torch.float16), lambda: ops.mx_dequantize(a, out=torch.empty(4, 63, device="cuda")),
        lambda: ops.mx_dequantize(a._replace(cols=200)), lambda: ops.mx_dequantize(a._replace(bits=4)),
        lambda: ops.mx_dequantize(a._replace(codes=a.codes[:, ::2])), lambda: ops.mx_dequantize(a._replace(scales=a.scales.cpu())),
        lambda: ops.mx_dequantize((a.codes, a.scales)),
        lambda: ops.mx_rmsnorm(x.bfloat16(), ones, 1e-6), lambda: ops.mx_rmsnorm(x, ones[:32], 1e-6),
        lambda: ops.mx_rmsnorm(x, ones.bfloat16(), 1e-6), lambda: ops.mx_rmsnorm(x, ones, 1e-6, delta=x[:2]),
        lambda: ops.mx_rmsnorm(x, ones, 1e-6, delta=x.half()), lambda: ops.mx_rmsnorm(x, ones, 1e-6, 6),
        lambda: ops.mx_rmsnorm(torch.zeros(1, 32769, device="cuda"), torch.ones(32769, device="cuda"), 1e-6),
        lambda: ops.mx_linear(a, a, out), lambda: ops.mx_linear(a, ops.mx_pack_linear(torch.randn(8, 65, device="cuda")), out),
        lambda: ops.mx_linear(a, w, out.bfloat16()), lambda: ops.mx_linear(a, w, out.T), lambda: ops.mx_linear(a, w, out[:3]),
        lambda: ops.mx_linear(a, w, out[:1].expand(4, 8)), lambda: ops.mx_linear(a, w, out.cpu()),
        lambda: ops.mx_rmsnorm(x[:1].expand(4, 64), ones, 1e-6, delta=x), lambda: ops.mx_dequantize(a, out=x[:1].expand(4, 64)),
        lambda: ops.mx_linear_glu(a, w, 8), lambda: ops.mx_linear_glu(a, glu, 129), lambda: ops.mx_linear_glu(a, glu, 0),
        lambda: ops.mx_linear_glu(a, glu, 8, 3), lambda: ops.mx_linear_glu(a, glu, 8, 8, out=a),
        lambda: ops.mx_pack_gate_up(torch.randn(8, 64, device="cuda"), torch.randn(9, 64, device="cuda")),
        lambda: ops.mx_linear(MxRows(a.codes, a.scales, 8, 64.0), w, out),
    ]
    before = x.clone()
    for i, call in enumerate(calls):
        with pytest.raises(KernelError):
            call()
            pytest.fail(f"call {i} was taken")
    fine(ops)
    assert torch.equal(x, before)

"""Matrices in four bits: making them, taking them back, and the products with them, against the format written out in 64 bits."""
import numpy as np
import pytest
import torch

import q4_helpers as q4
from velox_b200.csrc import ops

pytestmark = pytest.mark.gpu


def made(n, k, group, seed, dtype=torch.bfloat16):
    """(a matrix in four bits, what it stands for in 64 bits)"""
    g = torch.Generator().manual_seed(seed)
    w = (torch.randn(n, k, generator=g) * 0.02 * (0.5 + torch.rand(n, 1, generator=g))).to(dtype).cuda()
    m = ops.quantize_q4(w, group)
    return m, q4.matrix(*q4.unpack(m), group)


def rows_of(m, k, seed):
    g = torch.Generator().manual_seed(1000 + seed)
    x = torch.randn(m, k, generator=g)
    x[:, ::97] *= 8
    x = x.to(torch.bfloat16)
    return x.cuda(), x.to(torch.float64).numpy()


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,k", [(1, 128), (15, 384), (16, 1), (17, 5), (200, 1024)])
def test_quantize(n, k, group, dtype):
    k = k if k > 8 else k * group   # (an odd number of groups too)
    w = torch.randn(n, k, generator=torch.Generator().manual_seed(n + k)).mul_(0.02).to(dtype)
    m = ops.quantize_q4(w.cuda(), group)
    q, s, b = q4.quantise(w.float().numpy(), group)
    for got, want in zip(q4.unpack(m), (q, s, b)):
        assert np.array_equal(got, want)
    assert np.array_equal(ops.dequantize_q4(m).double().cpu().numpy(), q4.matrix(q, s, b, group))
    # within half a scale (and the scale's, the offset's and the value's roundings) of what was given
    limit = np.repeat(s, group, 1) * (0.5 + 15 * q4.HALF_BF16) + 2 * q4.HALF_BF16 * np.abs(np.repeat(b, group, 1)) + q4.HALF_BF16 * w.double().abs().numpy()
    assert (np.abs(q4.matrix(q, s, b, group) - w.double().numpy()) <= limit).all()


def test_padding_is_zero():
    m = ops.quantize_q4(torch.full((17, 96), 3.0, dtype=torch.bfloat16, device="cuda"), 32)
    codes, affine = m.codes, m.affine
    assert codes.shape == (2, 2, 4, 8, 2, 2) and affine.shape == (2, 4, 8, 2, 2)
    assert int(codes[1, :, :, 1:].abs().sum()) == 0 and float(affine[1, :, 1:].abs().sum()) == 0
    assert int(codes[:, 1, 2:].abs().sum()) == 0 and float(affine[:, 3].abs().sum()) == 0
    assert float(affine[1, :, 0, 1].abs().sum()) == 0


@pytest.mark.parametrize("group", [32, 64, 128])
def test_groups_at_the_edges_of_the_format(group):
    """Constant groups, zeros, tiny and huge values, ties, infinities and NaN: each in a group of its own, its neighbours untouched."""
    g = np.zeros((16, group), np.float32)
    g[0] = 0.37
    g[2] = np.linspace(0, 15, group)                     # scale 1, offset 0: codes with ties
    g[3] = np.where(np.arange(group) % 2, 0.5, 15.0)
    g[3, 0] = 0.0
    g[4] = 1e-39 * np.arange(group)
    g[5] = 3e38
    g[5, 1] = -3e38                                      # a range beyond float32
    g[6] = 1e38 * np.sin(np.arange(group))
    g[7, 3] = np.nan
    g[8, 1] = np.inf
    g[9, 2] = -np.inf
    g[10] = -5.0
    g[10, 7] = -4.0
    g[11] = 1.0
    g[11, 5] = 1.0 + 2.0 ** -7
    w = np.concatenate([g, np.roll(g, 1, 0), g[::-1]], 1)
    m = ops.quantize_q4(torch.from_numpy(w).cuda(), group)
    want = q4.quantise(w, group)
    for got, x in zip(q4.unpack(m), want):
        assert np.array_equal(got, x, equal_nan=True)
    assert np.isnan(want[1][7, 0]) and np.isnan(want[1][5, 0]) and not np.isnan(want[1][6, 0])
    assert np.array_equal(ops.dequantize_q4(m).double().cpu().numpy(), q4.matrix(*want, group), equal_nan=True)


def test_quantize_rows_of_a_wider_matrix():
    w = torch.randn(33, 512, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).cuda()
    m = ops.quantize_q4(w[:, 64:320], 64)
    for got, want in zip(q4.unpack(m), q4.quantise(w[:, 64:320].float().cpu().numpy(), 64)):
        assert np.array_equal(got, want)


SIZES = [(1, 16, 64, 64), (1, 2048, 2048, 64), (2, 1, 32, 32), (3, 17, 96, 32), (5, 1000, 1056, 32), (8, 4096, 128, 128), (7, 40, 5120, 128),
         (8, 333, 4096, 64), (9, 100, 256, 64), (16, 130, 1024, 128), (17, 250, 2080, 32), (33, 129, 640, 64), (64, 512, 512, 64),
         (65, 1003, 1056, 32), (127, 256, 1984, 64), (128, 128, 4224, 128), (129, 200, 320, 64), (200, 2048, 2048, 64), (257, 144, 384, 128),
         (300, 15, 96, 32), (513, 700, 704, 64), (1025, 272, 256, 64),
         # matrices of many rows: blocks that form several tiles, two at a time (an odd number of them), by four warps
         (8, 5000, 96, 32), (3, 7201, 96, 32), (8, 7216, 576, 64), (1, 38000, 64, 64), (5, 37905, 224, 32), (12, 14401, 128, 128), (24, 7300, 160, 32),
         (32, 2000, 1024, 64), (20, 38016, 128, 64), (300, 4096, 512, 64), (700, 9001, 128, 128),
         # depths below a step, a single row of W, very many rows of x
         (40, 100, 32, 32), (33, 16, 64, 64), (1000, 30, 64, 32), (17, 1, 128, 128), (70001, 48, 64, 64)]


@pytest.mark.parametrize("m,n,k,group", SIZES)
@pytest.mark.parametrize("out_dtype,biased", [(torch.bfloat16, False), (torch.float32, True)])
def test_product(m, n, k, group, out_dtype, biased):
    w, w64 = made(n, k, group, m + n)
    x, x64 = rows_of(m, k, n)
    bias = torch.randn(n, generator=torch.Generator().manual_seed(5)).cuda() if biased else None
    got = ops.gemm_q4(x, w, bias, out_dtype)
    want = x64 @ w64.T + (bias.double().cpu().numpy() if biased else 0)
    assert got.dtype == out_dtype
    q4.close(got, want, q4.sum_bound(x64, w64) + (2.0 ** -23 * np.abs(want) if biased else 0), out_dtype)
    ops.check_device_errors()


@pytest.mark.parametrize("m,n,k,group", SIZES)
def test_gated(m, n, k, group):
    (gate, g64), (up, u64) = made(n, k, group, m), made(n, k, group, n + 7)
    x, x64 = rows_of(m, k, n + 1)
    name = sorted(ops.ACTIVATIONS)[(m + n) % len(ops.ACTIVATIONS)]
    got = ops.gated_q4(x, gate, up, name)
    want, bound = q4.gated(x64, g64, u64, name)
    q4.close(got, want, bound, torch.bfloat16)
    ops.check_device_errors()


@pytest.mark.parametrize("m,n,k,group", [(100, 300, 1056, 32), (270, 520, 1024, 128), (40, 2100, 640, 64)])
@pytest.mark.parametrize("columns", [16, 48, 112, 128, 256])
@pytest.mark.parametrize("splits", [1, 2, 3, 4, 8])
def test_tiles_of_the_tensor_core_product(m, n, k, group, columns, splits):
    """Every shape of a tile that the entry point takes, not only those that the sizes choose."""
    if splits > (k + 127) // 128:
        pytest.skip("more runs than steps are refused")
    (w, w64), (up, u64) = made(n, k, group, 3), made(n, k, group, 4)
    x, x64 = rows_of(m, k, 5)
    shape, error = ops.library().vx_gemm_q4_tc_shape, ops._error_address(x.device)
    out = torch.full((m, n), float("nan"), device="cuda")
    assert shape(x.data_ptr(), w.codes.data_ptr(), w.affine.data_ptr(), None, None, None, out.data_ptr(), m, n, k, k, n, group, 0, 0, 0, columns, splits,
                 error, ops._stream()) == 0
    q4.close(out, x64 @ w64.T, q4.sum_bound(x64, w64), torch.float32)
    if columns <= 128:
        out = torch.full((m, n), float("nan"), device="cuda", dtype=torch.bfloat16)
        assert shape(x.data_ptr(), w.codes.data_ptr(), w.affine.data_ptr(), up.codes.data_ptr(), up.affine.data_ptr(), None, out.data_ptr(), m, n, k, k, n,
                     group, ops.ACTIVATIONS["silu"], 1, 1, columns, splits, error, ops._stream()) == 0
        q4.close(out, *q4.gated(x64, w64, u64, "silu"), torch.bfloat16)
    ops.check_device_errors()


@pytest.mark.parametrize("m", [2, 16, 40])
def test_rows_behind_the_result_stay_as_they_were(m):
    """Odd numbers of columns, a result inside a wider tensor: nothing beside it is written."""
    n, k = 131, 192
    w, w64 = made(n, k, 64, 3)
    x, x64 = rows_of(m, k, 5)
    wide = torch.full((m + 2, n + 5), 7.0, device="cuda")
    inner = wide[1:m + 1, 2:n + 2]
    assert ops.library().vx_gemm_q4(x.data_ptr(), w.codes.data_ptr(), w.affine.data_ptr(), None, None, None, inner.data_ptr(), m, n, k, k, n + 5, 64, 0, 0, 0,
                                    ops._error_address(x.device), ops._stream()) == 0
    q4.close(inner, x64 @ w64.T, q4.sum_bound(x64, w64), torch.float32)
    wide[1:m + 1, 2:n + 2] = 7.0
    assert bool((wide == 7.0).all())


@pytest.mark.parametrize("m", [2, 40, 150])
@pytest.mark.parametrize("n", [131, 132])
@pytest.mark.parametrize("left,gap", [(2, 5), (1, 4), (2, 4), (1, 5)])
def test_bfloat16_results_inside_a_wider_tensor(m, n, left, gap):
    """Odd and even widths, distances and first elements: right inside, and nothing beside it is written."""
    k = 192
    (w, w64), (up, u64) = made(n, k, 64, 3), made(n, k, 64, 4)
    x, x64 = rows_of(m, k, 5)
    lib, error = ops.library(), ops._error_address(x.device)
    for second in (None, up):
        wide = torch.full((m + 2, n + gap), 7.0, device="cuda", dtype=torch.bfloat16)
        inner = wide[1:m + 1, left:n + left]
        assert lib.vx_gemm_q4(x.data_ptr(), w.codes.data_ptr(), w.affine.data_ptr(), second and second.codes.data_ptr(), second and second.affine.data_ptr(),
                              None, inner.data_ptr(), m, n, k, k, n + gap, 64, ops.ACTIVATIONS["silu"], 1, 0, error, ops._stream()) == 0
        if second:
            q4.close(inner, *q4.gated(x64, w64, u64, "silu"), torch.bfloat16)
        else:
            q4.close(inner, x64 @ w64.T, q4.sum_bound(x64, w64), torch.bfloat16)
        wide[1:m + 1, left:n + left] = 7.0
        assert bool((wide == 7.0).all())
    ops.check_device_errors()


def test_two_streams_at_once():
    """Both kernels side by side with themselves: nothing is shared."""
    w, _ = made(2048, 2048, 64, 1)
    up, _ = made(2048, 2048, 64, 2)
    xs = [rows_of(m, 2048, m)[0] for m in (4, 90)]
    want = [(ops.gemm_q4(x, w, None, torch.float32), ops.gated_q4(x, w, up)) for x in xs]
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                got.append([(ops.gemm_q4(x, w, None, torch.float32), ops.gated_q4(x, w, up)) for x in xs])
    torch.cuda.synchronize()
    for g in got:
        for (a, b), (c, d) in zip(g, want):
            assert torch.equal(a, c) and torch.equal(b, d)
    ops.check_device_errors()


def test_offsets_beyond_32_bits():
    """1.2 million rows of 4,096: codes, dense values and results beyond 2^31 bytes and elements; the last rows are those of a small matrix."""
    n, k, tail = 1200000, 4096, 160
    codes = torch.zeros(n // 16, k // 64, 4, 8, 2, 2, dtype=torch.int32, device="cuda")
    affine = torch.zeros(n // 16, k // 64, 8, 2, 2, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    codes[-tail // 16:] = torch.randint(-2 ** 31, 2 ** 31 - 1, codes[-tail // 16:].shape, dtype=torch.int32, device="cuda", generator=g)
    affine[-tail // 16:] = (torch.rand(affine[-tail // 16:].shape, device="cuda", generator=g) * 0.01).to(torch.bfloat16)
    big = ops.Q4Matrix(codes, affine, n, k, 64)
    small = ops.Q4Matrix(codes[-tail // 16:].clone(), affine[-tail // 16:].clone(), tail, k, 64)
    w64 = q4.matrix(*q4.unpack(small), 64)
    for m in (1, 40):
        x, x64 = rows_of(m, k, m)
        got = ops.gemm_q4(x, big, None, torch.float32)
        q4.close(got[:, -tail:], x64 @ w64.T, q4.sum_bound(x64, w64), torch.float32)
        assert float(got[:, :-tail].abs().max()) == 0.0
        del got
    dense = ops.dequantize_q4(big)
    assert np.array_equal(dense[-tail:].double().cpu().numpy(), w64) and float(dense[:-tail].abs().max()) == 0.0
    del big, codes, affine
    again = ops.quantize_q4(dense, 64)
    want = ops.quantize_q4(dense[-tail:], 64)
    assert torch.equal(again.codes[-tail // 16:], want.codes) and torch.equal(again.affine[-tail // 16:], want.affine)
    ops.check_device_errors()


@pytest.mark.parametrize("name", sorted(ops.ACTIVATIONS))
@pytest.mark.parametrize("m", [4, 40])
def test_every_activation(m, name):
    (gate, g64), (up, u64) = made(96, 256, 64, 1), made(96, 256, 64, 2)
    x, x64 = rows_of(m, 256, 3)
    x, x64 = x * 8, x64 * 8
    want, bound = q4.gated(x64, g64, u64, name)
    q4.close(ops.gated_q4(x, gate, up, name), want, bound, torch.bfloat16)


def odd_matrix(n, k, group, seed):
    """Scales and offsets of every size and sign: zero, subnormal, at both ends of those that are raised by 2^133, large; mixed within a row,
    a tile and a warp."""
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(-2 ** 31, 2 ** 31 - 1, (-(-n // 16), -(-k // 64), 4, 8, 2, 2), generator=g, dtype=torch.int32)
    bits = torch.tensor([0x0000, 0x0001, 0x007f, 0x0080, 0x00ff, 0x3c00, 0x3cff, 0x3d00, 0x3d01, 0x3f80, 0x4300, 0x8000, 0xbc00, 0xbf80], dtype=torch.int32)
    shape = (-(-n // 16), -(-k // 64) * 64 // group, 8, 2, 2)
    affine = bits[torch.randint(0, len(bits), shape, generator=g)]
    affine[..., 1] = bits[torch.randint(5, len(bits), shape[:-1], generator=g)]
    plain = torch.rand(shape[:2], generator=g) < 0.5     # half of the groups of a tile: scales as trained matrices have them
    affine[..., 0][plain] = 0x3c10
    return ops.Q4Matrix(codes.cuda(), affine.to(torch.int16).view(torch.bfloat16).cuda(), n, k, group)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,n,k", [(1, 64, 512), (8, 7300, 384), (13, 100, 1152), (30, 50, 640), (70, 200, 896), (5, 38000, 256)])
def test_scales_and_offsets_of_every_size(m, n, k, group):
    w, up = odd_matrix(n, k, group, m), odd_matrix(n, k, group, m + 1)
    w64, u64 = (q4.matrix(*q4.unpack(v), group) for v in (w, up))
    assert np.array_equal(ops.dequantize_q4(w).double().cpu().numpy(), w64)
    x, x64 = rows_of(m, k, n)
    q4.close(ops.gemm_q4(x, w, None, torch.float32), x64 @ w64.T, q4.sum_bound(x64, w64), torch.float32)
    want, bound = q4.gated(x64, w64, u64, "relu")
    q4.close(ops.gated_q4(x, w, up, "relu"), want, bound, torch.bfloat16)
    ops.check_device_errors()


def test_product_is_that_of_the_dense_matrix():
    """The same matrix, dense and in four bits, through the engine's products: float32 sums of the same terms."""
    w, w64 = made(256, 512, 64, 9)
    x, x64 = rows_of(8, 512, 9)
    dense = ops.gemm_bf16(x, ops.dequantize_q4(w), None, torch.float32).double().cpu().numpy()
    got = ops.gemm_q4(x, w, None, torch.float32).double().cpu().numpy()
    assert (np.abs(dense - got) <= 2 * q4.sum_bound(x64, w64)).all()


def test_a_rows_result_does_not_depend_on_its_neighbours():
    w, _ = made(300, 1024, 64, 4)
    up, _ = made(300, 1024, 64, 5)
    x, _ = rows_of(8, 1024, 4)
    whole, pair = ops.gemm_q4(x, w), ops.gated_q4(x, w, up)
    for m in range(1, 8):
        assert torch.equal(ops.gemm_q4(x[:m], w), whole[:m])
        assert torch.equal(ops.gated_q4(x[m:], w, up), pair[m:])


@pytest.mark.parametrize("m", [4, 70, 300])
def test_the_same_result_every_time(m):
    w, _ = made(512, 2048, 64, 4)
    x, _ = rows_of(m, 2048, 4)
    first = ops.gemm_q4(x, w, None, torch.float32)
    for _ in range(5):
        assert torch.equal(ops.gemm_q4(x, w, None, torch.float32, w_ready=True), first)


@pytest.mark.parametrize("m", [6, 50, 150])
def test_values_that_are_not_finite_stay_in_their_rows(m):
    w, w64 = made(64, 256, 64, 4)
    x, x64 = rows_of(m, 256, 4)
    x[1, 5] = float("nan")
    x[3, 200] = float("inf")
    got = ops.gemm_q4(x, w, None, torch.float32)
    good = [i for i in range(m) if i not in (1, 3)]
    q4.close(got[good], (x64 @ w64.T)[good], q4.sum_bound(x64[good], w64), torch.float32)
    assert bool(got[1].isnan().all()) and not bool(got[3].isfinite().any())
    # a group of W that stands for NaN: its row of W, that column of the result
    dense = torch.randn(64, 256, generator=torch.Generator().manual_seed(8)).to(torch.bfloat16).cuda()
    dense[7, 9] = float("inf")
    bad = ops.gemm_q4(rows_of(m, 256, 5)[0], ops.quantize_q4(dense, 64), None, torch.float32)
    assert bool(bad[:, 7].isnan().all()) and bool(bad[:, :7].isfinite().all()) and bool(bad[:, 8:].isfinite().all())


@pytest.mark.parametrize("m", [0, 1, 5, 40, 150])
def test_rows_of_a_wider_tensor_and_none(m):
    w, w64 = made(100, 320, 64, 6)
    wide, _ = rows_of(max(m, 2), 400, 6)
    x = wide[:m, 8:328]
    got = ops.gemm_q4(x, w, None, torch.float32)
    x64 = x.double().cpu().numpy()
    q4.close(got, x64 @ w64.T, q4.sum_bound(x64, w64), torch.float32)
    assert ops.gated_q4(x, w, w).shape == (m, 100)
    if m == 1:   # (a lone row's stride says nothing)
        assert torch.equal(ops.gemm_q4(x.as_strided((1, 320), (3, 1)), w, None, torch.float32), got)


@pytest.mark.parametrize("m", [3, 90])
def test_on_another_stream_and_in_a_graph(m):
    w, _ = made(256, 512, 64, 7)
    up, _ = made(256, 512, 64, 8)
    x, _ = rows_of(m, 512, 7)
    y, _ = rows_of(m, 512, 70)
    want = [(ops.gemm_q4(v, w, None, torch.float32), ops.gated_q4(v, w, up)) for v in (x, y)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.gemm_q4(x, w, None, torch.float32), ops.gated_q4(x, w, up)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0][0]) and torch.equal(got[1], want[0][1])
    fed = x.clone()
    graphs = []
    for _ in range(2):   # (two captures share nothing)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            h = ops.gated_q4(fed, w, up, w_ready=True)
            out = ops.gemm_q4(fed, w, None, torch.float32, w_ready=True), h
        graphs.append((graph, out))
    for v, (a, b) in ((y, want[1]), (x, want[0])):
        fed.copy_(v)
        for graph, out in graphs:
            graph.replay()
        for graph, out in graphs:
            assert torch.equal(out[0], a) and torch.equal(out[1], b)
    ops.check_device_errors()


@pytest.mark.parametrize("m", [2, 70])
def test_a_matrix_made_just_before(m):
    """Without `w_ready` nothing of the matrix is read before the kernel that makes it has ended."""
    x, x64 = rows_of(m, 1024, 1)
    for seed in range(20):
        dense = torch.randn(640, 1024, device="cuda").to(torch.bfloat16)
        w = ops.quantize_q4(dense, 64)
        got = ops.gemm_q4(x, w, None, torch.float32)
        w64 = q4.matrix(*q4.unpack(w), 64)
        q4.close(got, x64 @ w64.T, q4.sum_bound(x64, w64), torch.float32)


def test_refusals():
    w, _ = made(32, 128, 64, 1)
    x, _ = rows_of(2, 128, 1)
    for call, why in [
            (lambda: ops.gemm_q4(x.float(), w), "bfloat16 a"), (lambda: ops.gemm_q4(x[:, :64], w), "bfloat16 a"),
            (lambda: ops.gemm_q4(x[0], w), "bfloat16 a"), (lambda: ops.gemm_q4(x, w, None, torch.float16), "bfloat16 or float32 out"),
            (lambda: ops.gemm_q4(rows_of(2, 132, 1)[0][:, :128], w), "16-byte aligned"),
            (lambda: ops.gemm_q4(rows_of(2, 136, 1)[0][:, 1:129], w), "16-byte aligned"),
            (lambda: ops.gemm_q4(rows_of(128, 2, 1)[0].t(), w), "contiguous"),
            (lambda: ops.gemm_q4(x[:1].expand(3, 128), w), "contiguous"),
            (lambda: ops.gemm_q4(x, w, torch.zeros(31, device="cuda")), "bias"),
            (lambda: ops.gemm_q4(x, w, torch.zeros(32, device="cuda", dtype=torch.bfloat16)), "bias"),
            (lambda: ops.gemm_q4(x, w, torch.zeros(64, device="cuda")[::2]), "bias"),
            (lambda: ops.gemm_q4(x.cpu(), w), "CUDA tensors"),
            (lambda: ops.gated_q4(x, w, w, "swish"), "unknown activation"),
            (lambda: ops.gated_q4(x, w, made(33, 128, 64, 1)[0]), "one shape"), (lambda: ops.gated_q4(x, w, made(32, 128, 32, 1)[0]), "one shape"),
            (lambda: ops.quantize_q4(x.half(), 64), "bfloat16 or float32"), (lambda: ops.quantize_q4(x, 48), "groups of"),
            (lambda: ops.quantize_q4(x[:, :96], 64), "multiple of the group"), (lambda: ops.quantize_q4(x[:0], 64), "positive"),
            (lambda: ops.quantize_q4(x[:, 1:65], 64), "aligned"), (lambda: ops.quantize_q4(x.t(), 64), "contiguous")]:
        with pytest.raises(ops.KernelError, match=why):
            call()


@pytest.mark.parametrize("group", [32, 64, 128])
def test_groups_that_fill_the_range_of_float32(group):
    """max - min just below float32's largest: w - b may overflow where b is the minimum rounded away, and the largest value's code is 15 all the same."""
    n = 96
    g = torch.Generator().manual_seed(group)
    u = torch.rand(n, group, generator=g).numpy()
    span = np.linspace(3.36e38, 3.4028e38, n)[:, None]
    low = -span * np.linspace(0.5, 0.503, 7)[np.arange(n) % 7][:, None]
    u[:, 1], u[:, group - 2] = 0, 1
    w = (low + span * u).astype(np.float32)
    w[0] = -1.709387e38
    w[0, 5:] = np.float32(1.693113e38)
    want = q4.quantise(w, group)
    top = np.isfinite(want[1][:, 0])
    with np.errstate(over="ignore"):
        overflows = top & ~np.isfinite(w.max(1) - want[2][:, 0].astype(np.float32))
    assert top[0] and overflows[0] and overflows.sum() >= 4 and (top & ~overflows).sum() >= 4
    assert (want[0][np.arange(n), w.argmax(1)][top] == 15).all()
    for got, x in zip(q4.unpack(ops.quantize_q4(torch.from_numpy(w).cuda(), group)), want):
        assert np.array_equal(got, x, equal_nan=True)


@pytest.mark.parametrize("m,n,k,plain,gated", [(16, 9000, 4096, 0, 0), (17, 512, 512, 0, 0), (32, 4096, 4096, 0, 1), (32, 1000, 2048, 0, 0), (17, 9000, 4096, 1, 1),
                                               (33, 64, 64, 1, 1)])
def test_the_products_that_wait_are_counted(m, n, k, plain, gated):
    """A launch is counted as one with bounded waits where the kernel that ran has them, through the call module and without it."""
    w = ops.quantize_q4(torch.zeros(n, k, dtype=torch.bfloat16, device="cuda"), 64)
    x, _ = rows_of(m, k, 1)
    ways = {False: [lambda: ops.gemm_q4(x, w), lambda: ops._q4_product("gemm_q4", x, w, None, None, torch.bfloat16, 0, False)],
            True: [lambda: ops.gated_q4(x, w, w), lambda: ops._q4_product("gated_q4", x, w, w, None, torch.bfloat16, 0, False)]}
    for pair, calls in ways.items():
        for call in calls:
            before = ops.bounded_wait_launches()
            call()
            assert ops.bounded_wait_launches() - before == (gated if pair else plain)
    ops.check_device_errors()


@pytest.mark.parametrize("m,n,k,group", [(9, 2400, 4096, 32), (12, 15000, 160, 32), (16, 7000, 1056, 32), (24, 15001, 160, 32), (32, 40000, 96, 32), (12, 40003, 96, 32),
                                         (10, 15000, 320, 64), (24, 15001, 384, 128)])
def test_blocks_that_have_one_buffer_for_their_sums(m, n, k, group):
    """9 to 32 rows, matrices of so many rows that a block forms several tiles: with small groups its sums are held once, and what one tile's epilogue
    reads is not overwritten by the next tile."""
    (w, w64), (up, u64) = made(n, k, group, 21), made(n, k, group, 22)
    x, x64 = rows_of(m, k, 23)
    q4.close(ops.gemm_q4(x, w, None, torch.float32), x64 @ w64.T, q4.sum_bound(x64, w64), torch.float32)
    q4.close(ops.gated_q4(x, w, up, "silu"), *q4.gated(x64, w64, u64, "silu"), torch.bfloat16)


@pytest.mark.parametrize("m,n,k,group", [(1, 96, 12288, 64), (8, 200, 17408, 128), (16, 64, 18432, 32), (24, 100, 12288, 64), (40, 130, 12288, 64), (200, 256, 17408, 128),
                                         (700, 40, 25600, 64)])
def test_deep_products(m, n, k, group):
    """As deep as the way down of a feed-forward and deeper, within a bound that a lost block of k, or sums held in fewer bits, would break."""
    (w, w64), (up, u64) = made(n, k, group, 31), made(n, k, group, 32)
    x, x64 = rows_of(m, k, 33)
    bound = q4.run_bound(x64, w64)
    want = x64 @ w64.T
    assert np.median(bound) < 2e-3 * np.abs(want).mean()
    q4.close(ops.gemm_q4(x, w, None, torch.float32), want, bound, torch.float32)
    q4.close(ops.gemm_q4(x, w), want, bound, torch.bfloat16)
    q4.close(ops.gated_q4(x, w, up, "silu"), *q4.gated(x64, w64, u64, "silu", q4.run_bound), torch.bfloat16)
    ops.check_device_errors()


def test_results_of_more_than_31_bits_of_elements():
    """2,000 rows by 1.2 million columns: the last rows and columns are those of a small product."""
    m, n, k, tail = 2000, 1200000, 64, 160
    assert m * n > 2 ** 31
    codes = torch.zeros(n // 16, 1, 4, 8, 2, 2, dtype=torch.int32, device="cuda")
    affine = torch.zeros(n // 16, 1, 8, 2, 2, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(2)
    codes[-tail // 16:] = torch.randint(-2 ** 31, 2 ** 31 - 1, codes[-tail // 16:].shape, dtype=torch.int32, device="cuda", generator=g)
    affine[-tail // 16:] = (torch.rand(affine[-tail // 16:].shape, device="cuda", generator=g) * 0.01).to(torch.bfloat16)
    big = ops.Q4Matrix(codes, affine, n, k, 64)
    w64 = q4.matrix(*q4.unpack(ops.Q4Matrix(codes[-tail // 16:].clone(), affine[-tail // 16:].clone(), tail, k, 64)), 64)
    x, x64 = rows_of(m, k, 4)
    for out_dtype in (torch.bfloat16, torch.float32):
        got = ops.gemm_q4(x, big, None, out_dtype)
        q4.close(got[:, -tail:], x64 @ w64.T, q4.sum_bound(x64, w64), out_dtype)
        assert not bool(got[:, :-tail].any())
        del got
    got = ops.gated_q4(x, big, big)
    q4.close(got[:, -tail:], *q4.gated(x64, w64, w64, "silu"), torch.bfloat16)
    assert not bool(got[:, :-tail].any())
    ops.check_device_errors()


@pytest.mark.parametrize("m", [8, 14, 40])
def test_rows_that_lie_far_apart(m):
    """Rows of x, and of a result inside a wider tensor, whose offsets pass 31 bits of elements."""
    n, k, group = 200, 320, 64
    far = (2 ** 31 // (m - 1) + 64) // 8 * 8
    assert (m - 1) * far > 2 ** 31 and far < 2 ** 31
    (w, w64), (up, u64) = made(n, k, group, 41), made(n, k, group, 42)
    x, x64 = rows_of(m, k, 43)
    apart = torch.zeros((m - 1) * far + k, dtype=torch.bfloat16, device="cuda").as_strided((m, k), (far, 1))
    apart.copy_(x)
    q4.close(ops.gemm_q4(apart, w, None, torch.float32), x64 @ w64.T, q4.sum_bound(x64, w64), torch.float32)
    q4.close(ops.gated_q4(apart, w, up), *q4.gated(x64, w64, u64, "silu"), torch.bfloat16)
    del apart
    lib, error = ops.library(), ops._error_address(x.device)
    wide = torch.zeros((m - 1) * far + n, dtype=torch.bfloat16, device="cuda")
    for second in (None, up):
        assert lib.vx_gemm_q4(x.data_ptr(), w.codes.data_ptr(), w.affine.data_ptr(), second and second.codes.data_ptr(), second and second.affine.data_ptr(), None,
                              wide.data_ptr(), m, n, k, k, far, group, ops.ACTIVATIONS["silu"], 1, 0, error, ops._stream()) == 0
        inner = wide.as_strided((m, n), (far, 1))
        if second:
            q4.close(inner, *q4.gated(x64, w64, u64, "silu"), torch.bfloat16)
        else:
            q4.close(inner, x64 @ w64.T, q4.sum_bound(x64, w64), torch.bfloat16)
        inner.zero_()
        assert not bool(wide.any())
    ops.check_device_errors()


def test_beside_the_dense_product_on_another_stream():
    """Both products take tensor memory in clusters of blocks (24 rows: tiles of 16, k in four runs; dense: k in runs, two blocks an SM).  Their blocks never
    share an SM, so no cluster waits for the other's tensor memory."""
    w, _ = made(2048, 16384, 64, 1)
    x, _ = rows_of(24, 16384, 2)
    g = torch.Generator(device="cuda").manual_seed(3)
    dense = torch.randn(2048, 4096, generator=g, device="cuda").to(torch.bfloat16)
    y = torch.randn(24, 4096, generator=g, device="cuda").to(torch.bfloat16)
    want, also = ops.gemm_q4(x, w), ops.gemm_turned(y, dense, w_ready=True)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(40):
        with torch.cuda.stream(streams[0]):
            got.append(ops.gemm_q4(x, w, w_ready=True))
        with torch.cuda.stream(streams[1]):
            got += [ops.gemm_turned(y, dense, w_ready=True) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(v, also if i % 4 else want) for i, v in enumerate(got))
    ops.check_device_errors()

"""ternainfer_amd/int8_linear.py against the definition: integers and sums exactly, the three fp32 operations behind them too."""
import ctypes

import pytest
import torch

import ternainfer_amd as T
from ternainfer_amd import _lib
from tests import _drafting as P

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(shape, seed, dtype=torch.bfloat16):
    return torch.randn(shape, generator=_gen(seed), device="cuda").to(dtype)


def _int8(shape, seed, low=-128):
    return torch.randint(low, 128, shape, generator=_gen(seed), device="cuda", dtype=torch.int8)


def _scales(n, seed):
    return 0.001 + torch.rand(n, generator=_gen(seed), device="cuda")


def _say(*what):
    print("[case]", *what, flush=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("r,k", [(1, 1), (3, 16), (5, 17), (16, 64), (17, 128), (33, 129), (7, 1000), (4, 2560), (9, 6912), (2, 7169), (3, 20000), (2500, 40), (1, 131056)])
def test_rows_are_quantised(dtype, r, k):
    _say("quantise", dtype, r, k)
    x = _randn((r, k), 1, dtype)
    x[:, 0] *= 6
    got = T.quantise_rows(x)
    q, scale = P.quantise(x)
    assert (got.rows, got.columns) == (r, k) and torch.equal(P.unpack(got.packed, r, k), q) and torch.equal(got.scale, scale)


def test_rows_of_every_kind_are_quantised():
    x = _randn((12, 300), 2, torch.float32)
    x[0] = 0.0
    x[1, 5] = float("nan")
    x[2, 299] = float("inf")
    x[3, 0] = float("-inf")
    x[4] *= 2.0 ** -140                                                                   # below the normal numbers
    x[5] = 2.0 ** -121
    x[6] = torch.where(torch.arange(300, device="cuda") % 2 == 0, 2.0 ** -120, -2.0 ** -120)
    x[7, 17] = 3e38
    x[8] = torch.arange(300, device="cuda") - 127.0                                       # halves of a step
    x[9] = (torch.arange(300, device="cuda") % 255 - 127.0) / 2
    x[9, 0] = 127.0
    x[10] = -0.0
    for rows in (x, x.to(torch.bfloat16)):
        got, (q, scale) = T.quantise_rows(rows), P.quantise(rows)
        assert torch.equal(P.unpack(got.packed, 12, 300), q)
        assert torch.equal(got.scale.isnan(), scale.isnan()) and torch.equal(got.scale.nan_to_num(7.0), scale.nan_to_num(7.0))
        assert got.scale[[1, 2, 3]].isnan().all() and not q[[0, 1, 2, 3, 4, 5, 10]].any()


def test_rows_at_any_address():
    wide = _randn((20, 201), 3)
    for x in (wide[:, 1:], wide[:, 3:180], wide[::2, :200], wide.t().contiguous().t(), wide[:1].expand(20, 201), wide[:, :1], wide.float()[:, 1:], wide.view(-1)[5:].as_strided((10, 64), (201, 1))):
        got, (q, scale) = T.quantise_rows(x), P.quantise(x)
        assert torch.equal(P.unpack(got.packed, *x.shape), q) and torch.equal(got.scale, scale)
    ints = _int8((30, 211), 4)
    for x in (ints, ints[:, 1:], ints[:, 16:208], ints[::3, :7], ints.t().contiguous().t(), ints[:1].expand(9, 211)):
        scale = _scales(x.shape[0], 5)
        got = T.int8_rows(x, scale)
        assert torch.equal(P.unpack(got.packed, *x.shape), x) and torch.equal(got.scale, scale)


# one or more shapes of every tile, and of tiles in parts
SHAPES = [(1, 1, 1), (1, 2560, 640), (2, 17, 65), (16, 254, 16), (31, 100, 1000), (33, 33, 33), (60, 2560, 6912), (1, 300, 7000), (128, 2560, 6912), (64, 15, 8192), (333, 2501, 2000), (300, 300, 8192),
          (1, 50021, 640), (32, 60000, 200), (60, 50021, 128), (70, 40000, 130), (128, 13824, 640), (500, 2560, 352), (512, 13824, 130), (1000, 2560, 700), (2048, 3840, 260), (4096, 2560, 192),
          (1500, 20000, 64), (2049, 1025, 1001), (5000, 300, 100)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product(m, n, k):
    _say("product", m, n, k)
    x, w, xs, ws = _int8((m, k), 10), _int8((n, k), 11), _scales(m, 12), _scales(n, 13)
    rows, weight = T.int8_rows(x, xs), T.int8_rows(w, ws)
    for dtype in (torch.float32, torch.bfloat16):
        got = T.int8_linear(rows, weight, dtype)
        assert got.dtype == dtype and got.shape == (m, n) and got.is_contiguous()
        assert torch.equal(got, P.linear(x, xs, w, ws, dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n", [(3, n) for n in (*range(1, 20), 127, 129, 130, 255, 258, 260)] + [(1, 50021), (33, 60001), (64, 50022), (130, 13825), (512, 13826), (500, 6145), (4096, 2563), (2049, 4100), (1500, 20001)])
def test_results_of_rows_of_every_width(dtype, m, n):
    """Every element, and nothing in front of the results or behind them."""
    _say("width", dtype, m, n)
    k, size = 64, 2 if dtype == torch.bfloat16 else 4
    x, w, xs, ws = _int8((m, k), 14), _int8((n, k), 15), _scales(m, 16), _scales(n, 17)
    rows, weight, lib = T.int8_rows(x, xs), T.int8_rows(w, ws), _lib.load()
    room = torch.full((16 // size + m * n + 1024,), 7.0, dtype=dtype, device="cuda")
    p = lambda t, by=0: ctypes.c_void_p(t.data_ptr() + by)
    assert lib.ternaspmm_int8_linear(p(rows.packed), p(rows.scale), p(weight.packed), p(weight.scale), p(room, 16), int(dtype == torch.float32), None, m, n, k,
                                     ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
    got = room[16 // size:16 // size + m * n].view(m, n)
    assert torch.equal(got, P.linear(x, xs, w, ws, dtype)) and (room[:16 // size] == 7).all() and (room[16 // size + m * n:] == 7).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n,k", [(1, 100, 2560), (17, 257, 300), (65, 64, 6912), (400, 1000, 129)])
def test_product_of_rows_that_are_quantised_in_the_call(dtype, m, n, k):
    x, weight = _randn((m, k), 20, dtype), T.quantise_rows(_randn((n, k), 21, torch.float32))
    got = T.int8_linear(x, weight, torch.float32)
    (q, scale), w = P.quantise(x), P.unpack(weight.packed, n, k)
    assert torch.equal(got, P.linear(q, scale, w, weight.scale, torch.float32))
    assert torch.equal(got, T.int8_linear(T.quantise_rows(x), weight, torch.float32))
    assert torch.equal(T.int8_linear(x, weight), got.to(torch.bfloat16))
    assert torch.equal(T.int8_linear(torch.cat([x, x], 1)[:, :k], weight, torch.float32), got)


def test_more_than_two_to_the_31_results():
    m, n, k = 17000, 128257, 16
    _say("results", m, n, k)
    if torch.cuda.mem_get_info()[0] < 8 << 30:
        pytest.skip("4.4 GB of results")
    x, w, xs, ws = _int8((m, k), 60), _int8((n, k), 61), _scales(m, 62), _scales(n, 63)
    got = T.int8_linear(T.int8_rows(x, xs), T.int8_rows(w, ws))
    for at in (slice(0, 40), slice(16730, 16760), slice(m - 40, m)):                      # (row 16744 holds the 2^31st)
        assert torch.equal(got[at], P.linear(x[at], xs[at], w, ws, torch.bfloat16))


def test_many_rows():
    """Rows whose place is behind 2^31 bytes, in the tensor and packed."""
    r, k = 1 << 20, 2100
    _say("rows", r, k)
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("7 GB of rows")
    x = torch.zeros((r, k), dtype=torch.bfloat16, device="cuda")
    for at in (slice(0, 40), slice(r - 70, r)):
        x[at] = _randn((at.stop - at.start, k), 64)
    got = T.quantise_rows(x)
    band = 2 * ((k + 127) // 128) * 1024
    for first in (0, (r - 64) // 16):
        q, scale = P.quantise(x[16 * first:16 * first + 32])
        assert torch.equal(P.unpack(got.packed[first * band:(first + 2) * band], 32, k), q) and torch.equal(got.scale[16 * first:16 * first + 32], scale)
    ints = torch.zeros((r, k), dtype=torch.int8, device="cuda")
    ints[-33:] = _int8((33, k), 65)
    packed = T.int8_rows(ints, got.scale).packed
    assert torch.equal(P.unpack(packed[-3 * band:], 48, k), ints[-48:])


def test_the_largest_sums():
    """Every product 2^14, at the most columns: 2147221504, below 2^31."""
    k = 131056
    x = torch.full((3, k), -128, dtype=torch.int8, device="cuda")
    w = torch.cat([x[:2], -127 * torch.ones((1, k), dtype=torch.int8, device="cuda"), torch.full((1, k), 127, dtype=torch.int8, device="cuda")])
    one = torch.ones(4, device="cuda")
    got = T.int8_linear(T.int8_rows(x, one[:3]), T.int8_rows(w, one), torch.float32)
    assert torch.equal(got, torch.tensor([[k * 16384.0, k * 16384.0, k * 16256.0, k * -16256.0]], device="cuda").expand(3, 4))


def test_rows_that_are_not_finite_and_scales():
    x, weight = _randn((5, 200), 30), T.quantise_rows(_randn((70, 200), 31))
    x[1, 3], x[2, 4], x[3] = float("nan"), float("inf"), 0.0
    got = T.int8_linear(x, weight)
    assert got[1:3].isnan().all() and not got[3].any() and torch.isfinite(got[[0, 4]]).all()
    assert torch.equal(got[[0, 4]], T.int8_linear(x[[0, 4]], weight))
    broken = weight._replace(scale=torch.where(torch.arange(70, device="cuda") == 7, float("nan"), weight.scale))
    nan = T.int8_linear(x[:1], broken).isnan()[0]
    assert nan[7] and nan.sum() == 1


def test_refusals_and_no_rows():
    x, weight = _randn((4, 100), 40), T.quantise_rows(_randn((6, 100), 41))
    assert T.int8_linear(x[:0], weight).shape == (0, 6) and T.quantise_rows(x[:0]).packed.numel() == 0
    assert T.int8_linear(T.quantise_rows(x[:0]), weight).shape == (0, 6) and T.int8_linear(x, T.quantise_rows(x[:0])).shape == (4, 0)
    rows = T.quantise_rows(x)
    for call in (lambda: T.int8_linear(x[:, :99], weight), lambda: T.int8_linear(x.half(), weight), lambda: T.int8_linear(x[0], weight), lambda: T.int8_linear(x.cpu(), weight),
                 lambda: T.int8_linear(rows._replace(rows=17), weight), lambda: T.int8_linear(rows._replace(scale=rows.scale[:3]), weight), lambda: T.int8_linear(rows._replace(packed=rows.packed[16:]), weight),
                 lambda: T.int8_linear(rows._replace(scale=rows.scale.double()), weight), lambda: T.int8_linear(x, weight._replace(rows=40)), lambda: T.int8_linear(x, weight, torch.float16),
                 lambda: T.int8_linear(x, weight._replace(scale=weight.scale.cpu()))):
        with pytest.raises(ValueError, match="int8_linear"):
            call()
    for call in (lambda: T.quantise_rows(x.half()), lambda: T.quantise_rows(x[0]), lambda: T.quantise_rows(x[:, :0]), lambda: T.quantise_rows(_randn((1, 131057), 1))):
        with pytest.raises(ValueError, match="quantise_rows"):
            call()
    for call in (lambda: T.int8_rows(x, rows.scale), lambda: T.int8_rows(_int8((4, 5), 1), rows.scale[:3]), lambda: T.int8_rows(_int8((4, 5), 1), rows.scale.cpu()), lambda: T.int8_rows(_int8((4,), 1), rows.scale)):
        with pytest.raises(ValueError, match="int8_rows"):
            call()


def test_captured_and_on_another_stream():
    """A call in parts and one of a single launch, replayed with eager work between."""
    weights = [T.quantise_rows(_randn((2560, 6912), 50)), T.quantise_rows(_randn((300, 6912), 51))]
    x = _randn((60, 6912), 52)
    run = lambda: [T.int8_linear(x, w) for w in weights]
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
        with torch.cuda.graph(graph, stream=side):
            held = run()
    torch.cuda.current_stream().wait_stream(side)
    for i in range(4):
        x.copy_(_randn((60, 6912), 53 + i))
        want = run()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), i

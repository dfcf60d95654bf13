"""GPU tests of products in 8-bit integers (b2_int8_quantize, b2_int8_product) against plain implementations in 64 bits on the host."""
import math

import numpy as np
import pytest

from test_gpu_token_operators import TINY, TYPES, U, _close, _host, _out, _rand, _untouched, tm, u  # noqa: F401

pytestmark = pytest.mark.gpu


def _quantized(x):
    """integers and scales of the rows of x (64 bits on the host): the quotients are rounded to fp32, the product once"""
    most = np.abs(x).max(1).astype(np.float32)
    with np.errstate(divide="ignore", invalid="ignore"):
        inv = np.where(most > 2.0 ** -118, np.float32(127.0) / most, np.float32(0)).astype(np.float64)
    q = np.rint(x * inv[:, None])
    return q.astype(np.int64), np.where(most > 2.0 ** -118, most / np.float32(127.0), np.float32(0)).astype(np.float32)


def _int8(torch, rows, dim, seed, pad=0):
    """random integers over the whole range, rows at multiples of 16 bytes; what lies between the rows is not zero"""
    ld = (dim + 15) // 16 * 16 + pad
    g = torch.Generator().manual_seed(seed)
    full = torch.randint(-128, 128, (rows, ld), generator=g).to(torch.int8).cuda()
    return full[:, :dim]


@pytest.mark.parametrize("rows,dim,pad,shift", [(1, 1, 0, 0), (3, 5, 0, 1), (7, 16, 0, 0), (9, 259, 0, 0), (300, 40, 8, 0), (5, 1024, 0, 0), (4, 1279, 1, 3), (3, 4100, 0, 5), (2, 8192, 0, 0),
                                                (2, 9300, 3, 1), (2, 40001, 0, 0)])
@pytest.mark.parametrize("t", TYPES)
def test_quantize(tm, rows, dim, pad, shift, t):  # noqa: F811
    torch, b2 = tm
    x = _rand(torch, (rows, dim), t, rows + dim, 2.0, pad, shift)
    if rows > 2:
        x[1] = 0
        x[2, : dim // 2 + 1] *= 1e-3
    for ld in (dim, (dim + 15) // 16 * 16, dim + 3):
        full = torch.full((rows, ld), 55, dtype=torch.int8, device="cuda")
        q, s = full[:, :dim], torch.full((rows,), 7.0, device="cuda")
        b2.int8_quantize(q, s, x)
        want_q, want_s = _quantized(_host(x))
        assert np.array_equal(q.cpu().numpy(), want_q)
        assert np.array_equal(s.cpu().numpy(), want_s)
        assert (full[:, dim:] == 55).all()


def test_quantize_next_to_the_middle_of_two_integers(tm):  # noqa: F811
    """products that a rounding to fp32 would move onto the middle, or across it"""
    torch, b2 = tm
    r = np.random.default_rng(1)
    most = np.float32(r.uniform(0.5, 2.0, 400))
    inv = (np.float32(127.0) / most).astype(np.float64)
    half = (r.integers(-126, 126, (400, 63)) + 0.5) / inv[:, None]
    x = np.concatenate([most[:, None].astype(np.float64), half], 1).astype(np.float32)
    x[:, 1::2] = np.nextafter(x[:, 1::2], np.float32(9))
    xt = torch.from_numpy(x).cuda()
    q, s = torch.empty(400, 64, dtype=torch.int8, device="cuda"), torch.empty(400, device="cuda")
    b2.int8_quantize(q, s, xt)
    assert np.array_equal(q.cpu().numpy(), _quantized(x.astype(np.float64))[0])


@pytest.mark.parametrize("dim", [40, 3000, 20000])
def test_quantize_special_rows(tm, dim):  # noqa: F811
    torch, b2 = tm
    x = torch.ones(7, dim, device="cuda")
    x[0, dim // 2] = math.nan
    x[1, dim - 1] = math.inf
    x[2, 0] = -math.inf
    x[3] = 0
    x[3, 1] = -0.0
    x[4] = 2.0 ** -119                     # nothing above 2^-118
    x[5] = 2.0 ** -100
    x[6, 3] = -3.3e38
    q, s = torch.full((7, dim), 9, dtype=torch.int8, device="cuda"), torch.empty(7, device="cuda")
    b2.int8_quantize(q, s, x)
    assert torch.isnan(s[:3]).all() and (q[:5] == 0).all() and (s[3:5] == 0).all() and (q[5] == 127).all() and q[6, 3].item() == -127 and (q[6, 4:] == 0).all()
    # such rows in a product
    w, ws = _int8(torch, 9, dim, 3), torch.ones(9, device="cuda")
    out = torch.empty(7, 9, device="cuda")
    work = torch.empty(b2.int8_product_workspace(7, 9, dim), dtype=torch.uint8, device="cuda")
    b2.int8_product(out, x, w, ws, bias=torch.full((9,), 2.5, device="cuda"), workspace=work)
    assert torch.isnan(out[:3]).all() and (out[3:5] == 2.5).all() and torch.isfinite(out[5]).all()


# around the borders of a slab (128 positions), a tile (128 channels; 16 to 256 rows) and the ways in which a product is split
PRODUCTS = [(1, 1, 1), (1, 5, 16), (3, 130, 40), (8, 1000, 1024), (16, 127, 129), (17, 128, 128), (32, 300, 257), (33, 260, 511), (64, 129, 100), (65, 4000, 130), (128, 200, 1000), (129, 513, 384),
            (257, 385, 650), (300, 1030, 1), (1, 20000, 300), (520, 700, 2050), (2000, 33, 64), (700, 5000, 259), (5, 64, 8192), (40, 40, 100000), (600, 600, 131071),
            (300, 40000, 130), (1500, 8000, 1300), (513, 19000, 1152)]


@pytest.mark.parametrize("rows,channels,dim", PRODUCTS)
@pytest.mark.parametrize("o", TYPES)
def test_product_of_integers(tm, rows, channels, dim, o):  # noqa: F811
    torch, b2 = tm
    x, w = _int8(torch, rows, dim, 1, 16), _int8(torch, channels, dim, 2)
    if dim > 100000:
        x[0] = -128                        # the largest sums there are
        w[0] = -128
    g = torch.Generator().manual_seed(3)
    xs, ws, bias = (torch.rand(n, generator=g).cuda() + 0.1 for n in (rows, channels, channels))
    ws *= {"f32": 1.0, "bf16": 1.0, "f16": 1e-6}[o]
    full, out = _out(torch, (rows, channels), o, 3, 1)
    b2.int8_product(out, x, w, ws, bias=bias, x_scales=xs)
    total = x.double() @ w.double().t()    # whole numbers below 2^53
    s = xs.double()[:, None] * ws.double()
    want = _host(total * s + bias.double())
    # the sum's, the scales' and the product's roundings, then that of the sum with the bias
    _close(_host(out), want, 4 * u * _host((total * s).abs()) + (U[o] + u) * np.abs(want) + U[o] * 4 * u * _host((total * s).abs()) + TINY[o])
    _untouched(torch, full, out)
    if o == "f32":
        plain = torch.empty(rows, channels, device="cuda")
        one = torch.ones(rows, device="cuda")
        b2.int8_product(plain, x, w, torch.ones(channels, device="cuda"), x_scales=one)
        assert torch.equal(plain, total.float())                              # exact sums, rounded once


@pytest.mark.parametrize("rows,channels,dim", [(1, 3, 1), (4, 50, 259), (8, 3000, 1024), (20, 129, 77), (100, 300, 2000), (300, 500, 640), (2, 70, 9000), (1000, 129, 4100),
                                                (16, 5000, 2048), (9, 700, 1500), (32, 4000, 4096), (25, 1, 5000), (17, 12900, 2500), (16, 20000, 5000), (12, 37900, 600), (1, 1, 16000)])
@pytest.mark.parametrize("t,o", [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16"), ("f16", "f16")])
def test_product_of_activations(tm, rows, channels, dim, t, o):  # noqa: F811
    torch, b2 = tm
    x = _rand(torch, (rows, dim), t, dim, 1.5, 3, 1)
    w = _int8(torch, channels, dim, 2)
    ws = (torch.rand(channels, generator=torch.Generator().manual_seed(3)).cuda() + 0.1) * 1e-3
    work = torch.full((b2.int8_product_workspace(rows, channels, dim),), 0xA5, dtype=torch.uint8, device="cuda")
    full, out = _out(torch, (rows, channels), o, 0, 1)
    b2.int8_product(out, x, w, ws, workspace=work)
    q, s = _quantized(_host(x))
    want = (q.astype(np.float64) @ _host(w).T) * s.astype(np.float64)[:, None] * _host(ws)
    _close(_host(out), want, (U[o] + 4 * u) * np.abs(want) + TINY[o])
    _untouched(torch, full, out)
    # the two steps by themselves give the same bits
    rowb = (dim + 15) // 16 * 16
    xq, xs = torch.empty(rows, rowb, dtype=torch.int8, device="cuda")[:, :dim], torch.empty(rows, device="cuda")
    b2.int8_quantize(xq, xs, x)
    two = torch.empty(rows, channels, dtype=out.dtype, device="cuda")
    b2.int8_product(two, xq, w, ws, x_scales=xs)
    assert torch.equal(two, out)


def test_a_single_row_needs_no_pitch(tm):  # noqa: F811
    torch, b2 = tm
    x = torch.randint(-128, 128, (1, 41), dtype=torch.int8, device="cuda")
    w = torch.randint(-128, 128, (1, 41), dtype=torch.int8, device="cuda")
    out, one = torch.empty(1, 1, device="cuda"), torch.ones(1, device="cuda")
    b2.int8_product(out, x, w, one, x_scales=one)
    assert out.item() == (x.double() @ w.double().t()).item()


def test_products_in_turn_share_a_workspace(tm):  # noqa: F811
    """many products in a row, captured too: a product reads what its own quantisation wrote"""
    torch, b2 = tm
    rows, channels, dim = 24, 6000, 512
    xs = [_rand(torch, (rows, dim), "bf16", s, 1.0) for s in range(6)]
    w, ws = _int8(torch, channels, dim, 2), torch.rand(channels, device="cuda")
    work = torch.empty(b2.int8_product_workspace(rows, channels, dim), dtype=torch.uint8, device="cuda")
    outs = [torch.empty(rows, channels, device="cuda") for _ in xs]
    for x, o in zip(xs, outs):
        b2.int8_product(o, x, w, ws, workspace=work)
        torch.cuda.synchronize()
    want = [o.clone() for o in outs]
    for _ in range(30):
        for o in outs:
            o.zero_()
        for x, o in zip(xs, outs):
            b2.int8_product(o, x, w, ws, workspace=work)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
    st, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        for x, o in zip(xs, outs):
            b2.int8_product(o, x, w, ws, workspace=work, stream=st.cuda_stream)
    for _ in range(5):
        for o in outs:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.parametrize("dim", [60, 100, 200, 300, 400, 500, 640, 800, 1000, 1152, 1200])
def test_products_of_short_contractions_over_many_channels(tm, dim):  # noqa: F811
    """a pair of blocks has several tiles of channels, whose weights follow each other in the same place: one slab to ten of them"""
    torch, b2 = tm
    rows, channels = 300, 60001
    x, w = _int8(torch, rows, dim, 1), _int8(torch, channels, dim, 2)
    out = torch.empty(rows, channels, device="cuda")
    b2.int8_product(out, x, w, torch.ones(channels, device="cuda"), x_scales=torch.ones(rows, device="cuda"))
    assert torch.equal(out, (x.double() @ w.double().t()).float())


@pytest.mark.parametrize("rows,channels,dim", [(8, 5000, 700), (20, 1000, 4000), (700, 3000, 900), (400, 2000, 2000)])
def test_products_at_once(tm, rows, channels, dim):  # noqa: F811
    """on two streams, each with its own workspace, and in a graph with one for both in turn"""
    torch, b2 = tm
    xs = [_rand(torch, (rows, dim), "bf16", s, 1.0) for s in (1, 2)]
    w, ws = _int8(torch, channels, dim, 2), torch.rand(channels, device="cuda")
    work = [torch.empty(b2.int8_product_workspace(rows, channels, dim), dtype=torch.uint8, device="cuda") for _ in xs]
    outs = [torch.empty(rows, channels, device="cuda") for _ in xs]
    want = []
    for x, o, k in zip(xs, outs, work):
        b2.int8_product(o, x, w, ws, workspace=k)
        torch.cuda.synchronize()
        want.append(o.clone())
    streams = [torch.cuda.Stream() for _ in xs]
    for _ in range(20):
        for x, o, k, st in zip(xs, outs, work, streams):
            b2.int8_product(o, x, w, ws, workspace=k, stream=st.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=streams[0]):
        for x, o in zip(xs, outs):
            b2.int8_product(o, x, w, ws, workspace=work[0], stream=streams[0].cuda_stream)
    for o in outs:
        o.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_offsets_beyond_32_bits(tm):  # noqa: F811
    torch, b2 = tm
    dim, ld = 200, 1 << 30
    w = torch.empty(5 * ld, dtype=torch.int8, device="cuda").view(5, ld)[:, :dim]
    w.copy_(_int8(torch, 5, dim, 3))
    x = _int8(torch, 4, dim, 4)
    ones = torch.ones(5, device="cuda")
    out = torch.empty(4 * ((1 << 29) + 1), device="cuda").view(4, -1)[:, :5]        # 8.6 GB
    b2.int8_product(out, x, w, ones, x_scales=ones[:4])
    assert torch.equal(out, (x.double() @ w.double().t()).float())
    big = torch.empty(3 * ld, dtype=torch.bfloat16, device="cuda").view(3, ld)[:, :dim]
    big.copy_(_rand(torch, (3, dim), "bf16", 5))
    q = torch.empty(5 * ld, dtype=torch.int8, device="cuda").view(5, ld)[:3, :dim]
    s = torch.empty(3, device="cuda")
    b2.int8_quantize(q, s, big)
    assert np.array_equal(q.cpu().numpy(), _quantized(_host(big))[0])

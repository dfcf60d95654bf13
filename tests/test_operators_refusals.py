"""CPU tests of the boundary of the operators that answer with a token model and learn from another one (include/b2lstm.h: b2_distill_*, b2_beam_*,
b2_int8_*): what the Python binding and the library refuse before any work reaches a GPU.  The tensors are stand-ins with made-up addresses that nothing
may read."""
import pytest

import b2lstm
from test_operators_binding import Fake, FakeOn, refused

I32, U8, S8 = dict(dtype="torch.int32"), dict(dtype="torch.uint8"), dict(dtype="torch.int8")


def f(*s, **k):
    return Fake(*s, **k)


def test_distill_arguments():
    x, tok, lp, o = f(4, 16), f(4, 3, **I32), f(4, 3), f(4)
    call = b2lstm.distill_forward
    refused("null", call, None, tok, lp, o, o)
    refused("null", call, x, None, lp, o, o)
    refused("null", call, x, tok, lp, o, None)
    refused("not on the GPU", call, f(4, 16, cuda=False), tok, lp, o, o)
    refused("element type", call, f(4, 16, dtype="torch.float64"), tok, lp, o, o)
    refused("element type", call, x, f(4, 3, dtype="torch.int64"), lp, o, o)
    refused("element type", call, x, tok, f(4, 3, dtype="torch.bfloat16"), o, o)
    refused("shape", call, x, f(12, **I32), lp, o, o)
    refused("elements", call, x, tok, f(4, 2), o, o)
    refused("elements", call, x, f(3, 3, **I32), lp, o, o)
    refused("elements", call, x, tok, lp, f(5), o)
    refused("elements", call, x, tok, lp, o, o, lse_rest=f(3))
    refused("strides", call, f(4, 16, stride=(8, 1)), tok, lp, o, o)
    refused("error -1.*listed", call, x, f(4, 129, **I32), f(4, 129), o, o)
    refused("error -1.*listed", call, x, f(4, 0, **I32), f(4, 0), o, o)
    refused("error -5.*scale", call, x, tok, lp, o, o, scale=0.0)
    refused("error -5.*scale", call, x, tok, lp, o, o, scale=float("nan"))
    refused("error -5.*aligned", call, f(4, 16, address=4097), tok, lp, o, o)
    refused("error -5.*aligned", call, x, f(4, 3, address=4098, **I32), lp, o, o)
    refused("error -5.*aligned", call, x, tok, lp, o, o, lse_rest=f(4, address=4098))
    d, back = f(4, 16, address=8192), b2lstm.distill_backward
    refused("null", back, None, x, tok, lp, o, o)
    refused("null", back, d, x, tok, lp, o, None)
    refused("shape", back, f(4, 15), x, tok, lp, o, o)
    refused("element type", back, f(4, 16, dtype="torch.float16"), x, tok, lp, o, o)
    refused("error -5.*in place", back, f(4, 16, stride=(17, 1)), x, tok, lp, o, o)
    refused("error -5.*in place", back, x, x, tok, lp, o, o, accumulate=True)
    refused("error -5.*aligned", back, f(4, 16, address=8193), x, tok, lp, o, o)
    refused("error -5.*aligned", back, d, x, tok, lp, f(4, address=4098), o)


def test_select_arguments():
    x, sc, ts, tb = f(6, 16), f(6), f(2, 4), f(2, 4, **I32)
    ws = dict(workspace=f(1 << 20, **U8))
    call = b2lstm.beam_select
    refused("null", call, x, None, ts, tb, tb, **ws)
    refused("null", call, x, sc, ts, None, tb, **ws)
    refused("shape", call, x, sc, f(8), tb, tb, **ws)
    refused("rows of logits", call, x, sc, f(4, 4), tb, tb, **ws)
    refused("elements", call, x, f(5), ts, tb, tb, **ws)
    refused("elements", call, x, sc, ts, f(2, 3, **I32), tb, **ws)
    refused("element type", call, x, sc, ts, f(2, 4), tb, **ws)
    refused("elements", call, x, sc, ts, tb, tb, finished=f(5, **U8), **ws)
    refused("element type", call, x, sc, ts, tb, tb, finished=f(6), **ws)
    refused("elements", call, x, sc, ts, tb, tb, weights=f(2), **ws)
    refused("shape", call, x, sc, ts, tb, tb, mask=f(2, 16, **U8), **ws)
    refused("error -5.*null", call, x, sc, ts, tb, tb)
    refused("error -5.*16 bytes", call, x, sc, ts, tb, tb, workspace=f(1 << 20, address=4104, **U8))
    refused("error -1.*needed", call, x, sc, ts, tb, tb, workspace=f(64, **U8))
    refused("error -5.*end_token", call, x, sc, ts, tb, tb, finished=f(6, **U8), end_token=16, **ws)
    refused("error -5.*end_token", call, x, sc, ts, tb, tb, finished=f(6, **U8), end_token=-1, **ws)
    refused("end_token", call, x, sc, ts, tb, tb, end_token=1 << 40, **ws)
    refused("error -5.*scale", call, x, sc, ts, tb, tb, scale=float("inf"), **ws)
    refused("error -1.*continuations", call, x, sc, f(2, 65), f(2, 65, **I32), f(2, 65, **I32), **ws)
    refused("error -1.*beams", call, f(130, 16), f(130), ts, tb, tb, **ws)
    refused("error -5.*aligned", call, f(6, 16, address=4097), sc, ts, tb, tb, **ws)
    size = b2lstm.beam_select_workspace
    assert size(2, 65, 16, 4) == 0 and size(2, 3, 16, 65) == 0 and size(2, 3, (1 << 26) + 1, 4) == 0 and size(2, 0, 16, 4) == 0 and size(1 << 40, 3, 16, 4) == 0
    assert 0 < size(2, 3, 16, 4) < size(2, 3, 200000, 4)


def test_state_lists():
    class State(Fake):
        def element_size(self):
            return 4
    s = lambda *a, **k: State(*a, **k)  # noqa: E731
    parents = f(2, 3, **I32)
    refused("contiguous", b2lstm.StateList, [s(6, 4, stride=(8, 1))])
    refused("contiguous", b2lstm.StateList, [s(6, 4, cuda=False)])
    refused("no axis", b2lstm.StateList, [s(6, 4)], 2)
    refused("no axis", b2lstm.StateList, [s(6, 4)], -1)
    refused("1 tensors, 2 axes", b2lstm.StateList, [s(6, 4)], [0, 1])
    refused("2 outputs", b2lstm.StateList, [s(6, 4)], 0, [s(6, 4), s(6, 4)])
    refused("shape", b2lstm.StateList, [s(6, 4)], 0, [s(6, 5)])
    refused("element type", b2lstm.StateList, [s(6, 4)], 0, [s(6, 4, dtype="torch.float16")])
    refused("beams", b2lstm.StateList, [s(6, 4), s(4, 6)])
    refused("6 parents for 4 beams", b2lstm.beam_reorder, b2lstm.StateList([s(4, 4)]), parents)
    refused("shape", b2lstm.beam_reorder, b2lstm.StateList([s(6, 4)]), f(6, **I32))
    refused("element type", b2lstm.beam_reorder, b2lstm.StateList([s(6, 4)]), f(2, 3))
    refused("error -5.*overlap", b2lstm.beam_reorder, b2lstm.StateList([s(6, 4)], 0, [s(6, 4, address=4096 + 16)]), parents)
    refused("error -5.*null", b2lstm.beam_reorder, b2lstm.StateList([s(6, 4, address=0)]), parents)
    refused("error -1.*beams", b2lstm.beam_reorder, b2lstm.StateList([s(130, 4)]), f(2, 65, **I32))
    b2lstm.beam_reorder(b2lstm.StateList([]), f(2, 3, **I32))                       # nothing to do
    b2lstm.beam_reorder(b2lstm.StateList([s(0, 4, address=0)]), f(0, 3, address=0, **I32))


def test_int8_arguments():
    x, q, sc = f(4, 40), f(4, 40, stride=(48, 1), **S8), f(4)
    refused("null", b2lstm.int8_quantize, None, sc, x)
    refused("element type", b2lstm.int8_quantize, f(4, 40, **U8), sc, x)
    refused("element type", b2lstm.int8_quantize, q, sc, f(4, 40, **S8))
    refused("shape", b2lstm.int8_quantize, f(4, 41, **S8), sc, x)
    refused("elements", b2lstm.int8_quantize, q, f(5), x)
    refused("error -5.*aligned", b2lstm.int8_quantize, q, sc, f(4, 40, address=4098))
    w, wsc, out, ws = f(7, 40, stride=(48, 1), **S8), f(7), f(4, 7), dict(workspace=f(1 << 16, **U8))
    call = b2lstm.int8_product
    refused("null", call, None, x, w, wsc, **ws)
    refused("null", call, out, x, w, None, **ws)
    refused("shape", call, f(4, 8), x, w, wsc, **ws)
    refused("shape", call, out, f(4, 39), w, wsc, **ws)
    refused("element type", call, out, x, f(7, 40, **U8), wsc, **ws)
    refused("element type", call, f(4, 7, **S8), x, w, wsc, **ws)
    refused("element type", call, out, q, w, wsc, **ws)                           # int8 without its scales
    refused("element type", call, out, x, w, wsc, x_scales=sc, **ws)              # scales, but not int8
    refused("elements", call, out, x, w, f(6), **ws)
    refused("elements", call, out, x, w, wsc, bias=f(6), **ws)
    refused("error -5.*16 bytes", call, out, x, f(7, 40, **S8), wsc, **ws)
    refused("error -5.*16 bytes", call, out, x, f(7, 40, stride=(48, 1), address=4104, **S8), wsc, **ws)
    refused("error -5.*16 bytes", call, out, f(4, 40, **S8), w, wsc, x_scales=sc)
    refused("error -5.*workspace", call, out, x, w, wsc)
    refused("error -1.*needed", call, out, x, w, wsc, workspace=f(64, **U8))
    refused("error -5.*16 bytes", call, out, x, w, wsc, workspace=f(1 << 16, address=4104, **U8))
    refused("error -1.*positions", call, f(4, 7), f(4, 131072), f(7, 131072, **S8), wsc, **ws)
    size = b2lstm.int8_product_workspace
    assert size(4, 7, 131072) == 0 and size(-1, 7, 40) == 0 and size(4, 0, 40) == 0 and size(4, 7, 40) == 4 * 48 + 16


def test_calls_without_rows():
    e = dict(address=0)
    b2lstm.distill_forward(f(0, 16, **e), f(0, 3, **I32, **e), f(0, 3, **e), f(0, **e), f(0, **e))
    b2lstm.distill_backward(f(0, 16, **e), f(0, 16, **e), f(0, 3, **I32, **e), f(0, 3, **e), f(0, **e), f(0, **e))
    b2lstm.beam_select(f(0, 16, **e), f(0, **e), f(0, 4, **e), f(0, 4, **I32, **e), f(0, 4, **I32, **e))
    b2lstm.int8_quantize(f(0, 16, **S8, **e), f(0, **e), f(0, 16, **e))
    b2lstm.int8_product(f(0, 7, **e), f(0, 40, **e), f(7, 40, stride=(48, 1), **S8), f(7))


def test_addresses_and_distances_that_no_kernel_may_see():
    L, at = b2lstm.lib(), 4096
    assert L.b2_distill_forward(at, 0, 4, 16, 1 << 41, 1.0, at, at, 3, at, at, None, None) == -5
    assert L.b2_distill_forward(at, 0, 4, 16, 15, 1.0, at, at, 3, at, at, None, None) == -5
    assert L.b2_distill_forward(at, 0, 4, 16, 16, 1.0, at, at + 1, 3, at, at, None, None) == -5
    assert L.b2_distill_forward(at, 0, 4, (1 << 27) + 1, 1 << 28, 1.0, at, at, 3, at, at, None, None) == -1
    assert L.b2_distill_backward(at, 1 << 41, at, 0, 4, 16, 16, 1.0, at, at, 3, at, None, at, 0, None) == -5
    assert L.b2_beam_select(at, 0, 2, 3, 16, 1 << 41, None, 0, 1.0, at, None, None, 0, 4, at, at, at, at, 1 << 20, None) == -5
    assert L.b2_beam_select(at, 0, 2, 3, 16, 16, at, 15, 1.0, at, None, None, 0, 4, at, at, at, at, 1 << 20, None) == -5
    assert L.b2_beam_select(at, 0, 2, 3, 16, 16, None, 0, 1.0, at + 2, None, None, 0, 4, at, at, at, at, 1 << 20, None) == -5
    assert L.b2_int8_quantize(at, 15, at, at, 0, 4, 16, 16, None) == -5
    assert L.b2_int8_quantize(at, 16, at, at, 0, 4, 16, 1 << 41, None) == -5
    assert L.b2_int8_product(at, 0, 7, at, 3, 48, at, at, 1 << 40, at, None, 4, 7, 40, None, 0, None) == -5
    assert L.b2_int8_product(at, 3, 7, at, 3, 48, at, at, 48, at, None, 4, 7, 40, None, 0, None) == -5
    assert L.b2_int8_product(at, 0, 7, at, 0, 48, at, at, 48, at, None, 4, 7, 40, at, 1 << 16, None) == -5


def test_tensors_of_another_device():
    import ctypes as C
    from b2lstm import operators
    ops, library = operators._ops(), b2lstm.lib()
    real = {name: C.cast(getattr(library, name), C.c_void_p).value for name in operators._BOUND}
    current = C.CFUNCTYPE(C.c_int)(lambda: 1)                     # as if device 1 was the current one
    on = lambda d, *s, **k: FakeOn(d, *s, **k)  # noqa: E731
    try:
        ops.bind(dict(real, b2_current_device=C.cast(current, C.c_void_p).value), b2lstm.B2Error)
        refused("top_tokens is on device 0", b2lstm.distill_forward, on(1, 4, 16), on(0, 4, 3, **I32), on(1, 4, 3), on(1, 4), on(1, 4))
        refused("scores is on device 0", b2lstm.beam_select, on(1, 6, 16), on(0, 6), on(1, 2, 4), on(1, 2, 4, **I32), on(1, 2, 4, **I32))
        refused("q is on device 0", b2lstm.int8_quantize, on(0, 4, 40, **S8), on(1, 4), on(1, 4, 40))
        refused("w is on device 2", b2lstm.int8_product, on(1, 4, 7), on(1, 4, 40), on(2, 7, 40, **S8), on(1, 7))
        class State(FakeOn):
            def element_size(self):
                return 4
        refused("tensors are on device 0", b2lstm.beam_reorder, b2lstm.StateList([State(0, 6, 4)]), on(1, 2, 3, **I32))
        refused("devices", b2lstm.StateList, [State(0, 6, 4)], 0, [State(1, 6, 4, address=8192)])
    finally:
        ops.bind(real, b2lstm.B2Error)


def test_bytes_are_still_taken_for_masks_and_pattern_types():
    """int8, uint8 and bool all hold pattern types and masks"""
    for t in ("torch.int8", "torch.uint8", "torch.bool"):
        refused("error -5.*null", b2lstm.logprob_forward, f(4, 8), None, f(4), f(4), mask=f(8, dtype=t))
        refused("error -1.*at most", b2lstm.block_norm_forward, f(2, 8193), None, None, f(2, 8193, address=8192), pat_types=f(2, dtype=t))


if __name__ == "__main__":
    pytest.main([__file__])

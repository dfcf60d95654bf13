"""CPU tests of the token operators' boundary: what the Python binding and the library refuse before any work reaches a GPU.  The tensors are
stand-ins with made-up addresses that nothing may read."""
import ctypes as C

import pytest

import b2lstm


class Fake:
    def __init__(self, *shape, dtype="float32", stride=None, cuda=True, address=4096):
        self.shape, self.dtype, self.is_cuda, self.address = tuple(shape), dtype, cuda, address
        self._stride = stride

    def stride(self):
        if self._stride is not None:
            return self._stride
        out, n = [], 1
        for s in reversed(self.shape):
            out.insert(0, n)
            n *= s
        return tuple(out)

    def numel(self):
        n = 1
        for s in self.shape:
            n *= s
        return n

    def is_contiguous(self):
        return self._stride is None

    def data_ptr(self):
        return self.address


TOK = Fake(4, dtype="torch.int32")


def refused(text, fn, *a, **k):
    with pytest.raises(b2lstm.B2Error, match=text):
        fn(*a, **k)


def test_embedding_arguments():
    refused("shape", b2lstm.embedding_forward, Fake(3, 8), Fake(10, 8), TOK)
    refused("shape", b2lstm.embedding_forward, Fake(32), Fake(10, 8), TOK)
    refused("not on the GPU", b2lstm.embedding_forward, Fake(4, 8, cuda=False), Fake(10, 8), TOK)
    refused("strides", b2lstm.embedding_forward, Fake(4, 8, stride=(16, 2)), Fake(10, 8), TOK)
    refused("strides", b2lstm.embedding_forward, Fake(4, 8, stride=(4, 1)), Fake(10, 8), TOK)
    refused("element type", b2lstm.embedding_forward, Fake(4, 8, dtype="torch.float64"), Fake(10, 8), TOK)
    refused("element type", b2lstm.embedding_forward, Fake(4, 8), Fake(10, 8), Fake(4, dtype="torch.int64"))
    refused("error -5.*aligned", b2lstm.embedding_forward, Fake(4, 8), Fake(10, 8, address=4098), TOK)
    refused("error -5.*null", b2lstm.embedding_forward, Fake(4, 8, address=0), Fake(10, 8), TOK)
    refused("error -1", b2lstm.embedding_forward, Fake(4, 1 << 21), Fake(10, 1 << 21), TOK)
    refused("no tensor", b2lstm.embedding_forward, Fake(4, 8), Fake(10, 8), [1, 2, 3, 4])
    with pytest.raises(TypeError):
        b2lstm.embedding_forward(Fake(4, 8), Fake(10, 8), TOK, scale="two")
    with pytest.raises(AttributeError):
        b2lstm.embedding_forward(object(), Fake(10, 8), TOK)
    refused("null", b2lstm.embedding_backward, Fake(10, 8), Fake(4, 8), TOK)
    refused("error -5.*256", b2lstm.embedding_backward, Fake(10, 8), Fake(4, 8), TOK, workspace=Fake(1 << 20, dtype="torch.uint8", address=64))
    refused("error -1.*needed", b2lstm.embedding_backward, Fake(10, 8), Fake(4, 8), TOK, workspace=Fake(16, dtype="torch.uint8"))
    assert b2lstm.embedding_backward_workspace(0, 10, 8) == 0 and b2lstm.embedding_backward_workspace(4, 0, 8) == 0
    assert b2lstm.embedding_backward_workspace(4, 10, 8) < b2lstm.embedding_backward_workspace(400000, 10, 8)


def test_logprob_arguments():
    f = lambda *s: Fake(*s)  # noqa: E731
    refused("error -5.*scale", b2lstm.logprob_forward, f(4, 8), TOK, f(4), f(4), scale=-1.0)
    refused("error -5.*scale", b2lstm.logprob_forward, f(4, 8), TOK, f(4), f(4), scale=float("inf"))
    refused("error -1.*alternatives", b2lstm.logprob_forward, f(4, 8), TOK, f(4), f(4), top_tokens=Fake(4, 40, dtype="torch.int32"), top_logprobs=f(4, 40))
    refused("error -5.*null", b2lstm.logprob_forward, f(4, 8), None, f(4), f(4))
    refused("elements", b2lstm.logprob_forward, f(4, 8), TOK, f(5), f(4))
    refused("shape", b2lstm.logprob_forward, f(4, 8), TOK, f(4), f(4), mask=Fake(3, 8, dtype="torch.bool"))
    refused("elements", b2lstm.logprob_forward, f(4, 8), TOK, f(4), f(4), mask=Fake(9, dtype="torch.bool"))
    refused("error -5.*in place", b2lstm.logprob_backward, Fake(4, 8, stride=(9, 1)), f(4, 8), TOK, f(4), f(4))
    refused("shape", b2lstm.logprob_backward, f(4, 9), f(4, 8), TOK, f(4), f(4))


def test_block_norm_arguments():
    x, o, st = Fake(4, 16), Fake(4, 16, address=8192), Fake(4, 4, address=16384)
    refused("error -1.*at most", b2lstm.block_norm_forward, Fake(2, 8193), None, None, Fake(2, 8193, address=8192))
    refused("error -1.*multiple", b2lstm.block_norm_forward, x, x, o, None, gate=Fake(3, 16))
    refused("error -5.*only y", b2lstm.block_norm_forward, x, o, o, None)
    refused("error -5.*statistics", b2lstm.block_norm_forward, x, None, None, o, stats=Fake(4, 4, address=16388))
    refused("element type", b2lstm.block_norm_forward, x, Fake(4, 16, dtype="torch.float16"), o, None)
    refused("elements", b2lstm.block_norm_forward, x, None, None, o, w_pre=Fake(15))
    refused("dy or dh", b2lstm.block_norm_backward, x, None, None, None, o, None, st)
    refused("without the gate", b2lstm.block_norm_backward, x, None, o, None, None, None, st, dgate=Fake(1, 16))
    refused("error -5.*same", b2lstm.block_norm_backward, x, x, o, None, None, o, st, workspace=Fake(1 << 24, dtype="torch.uint8"))
    assert b2lstm.block_norm_backward_workspace(0, 16) == 0 and b2lstm.block_norm_backward_workspace(5, 9000) == 0


def test_tensor_lists():
    ws = Fake(1 << 16, dtype="torch.uint8")
    refused("2 tensors and 1 outputs", b2lstm.TensorList, [Fake(3), Fake(3)], [Fake(3)])
    refused("element type", b2lstm.TensorList, [Fake(3, dtype="torch.int32")])
    refused("contiguous", b2lstm.TensorList, [Fake(3, 3, stride=(1, 3))])
    refused("error -5.*null pointer", b2lstm.gradient_norm, b2lstm.TensorList([Fake(3, address=0)]), Fake(1), workspace=ws)
    refused("error -5.*aligned", b2lstm.gradient_norm, b2lstm.TensorList([Fake(3, address=4098)]), Fake(1), workspace=ws)
    refused("error -1.*elements", b2lstm.gradient_clip, b2lstm.TensorList([Fake(3)], [Fake(4, address=8192)]), 1.0, Fake(1), workspace=ws)
    refused("error -5.*another element type", b2lstm.gradient_clip, b2lstm.TensorList([Fake(3)], [Fake(3, dtype="torch.bfloat16")]), 1.0, Fake(1), workspace=ws)
    refused("error -5.*largest norm", b2lstm.gradient_clip, b2lstm.TensorList([Fake(3)]), float("nan"), Fake(1), workspace=ws)
    refused("error -1.*needed", b2lstm.gradient_clip, b2lstm.TensorList([Fake(3)]), 1.0, Fake(1), workspace=Fake(8, dtype="torch.uint8"))


def test_addresses_and_distances_that_no_kernel_may_see():
    L, at = b2lstm.lib(), 4096
    assert L.b2_logprob_forward(at, 0, 4, 16, 16, None, 0, 1.0, at + 2, at, at, None, 0, None, None, None) == -5
    assert L.b2_logprob_forward(at, 0, 4, 16, 16, None, 0, 1.0, at, at, at + 1, None, 0, None, None, None) == -5
    assert L.b2_logprob_forward(at, 0, 4, 16, 1 << 41, None, 0, 1.0, at, at, at, None, 0, None, None, None) == -5
    assert L.b2_logprob_forward(at, 0, 4, 16, 16, at, 1 << 41, 1.0, at, at, at, None, 0, None, None, None) == -5
    assert L.b2_logprob_backward(at, 1 << 41, at, 0, 4, 16, 16, None, 0, 1.0, at, at, at, None, None, None) == -5
    assert L.b2_logprob_backward(at, 16, at, 0, 4, 16, 16, None, 0, 1.0, at, at + 2, at, None, None, None) == -5
    assert L.b2_embedding_forward(at, 0, 1 << 41, at, 0, 16, 4, 16, at, 4, 1.0, None) == -5
    assert L.b2_embedding_forward(at, 0, 16, at, 0, 16, 4, 16, at + 1, 4, 1.0, None) == -5
    assert L.b2_embedding_backward(at, 0, 16, 4, 16, at, 0, 1 << 41, at, 4, 1.0, 0, at, 1 << 20, None) == -5
    assert L.b2_gradient_norm(None, 0, at + 2, at, 1 << 20, None) == -5


def test_the_net_refuses_a_clipping_without_a_net():
    assert b2lstm.lib().b2_net_set_gradient_clipping(None, 1.0) == -5
    assert b2lstm.lib().b2_net_gradient_norm(None, C.byref(C.c_float())) == -5


def test_the_workspace_of_sizes_that_the_norm_gradient_refuses():
    """a gate with more rows than there are frames, or with rows that the frames are no multiple of (the plan of such a call would divide by zero)"""
    size = b2lstm.block_norm_backward_workspace
    assert size(4, 8, 100) == 0 and size(5, 8, 3) == 0 and size(1, 8, 2 ** 40) == 0
    assert size(6, 8, 3) > 0 and size(6, 8, 6) > 0 and size(6, 8) > 0


class FakeOn(Fake):
    """one that knows its device, as torch's tensors do"""

    def __init__(self, device, *shape, **k):
        super().__init__(*shape, **k)
        self.device = device

    def get_device(self):
        return self.device


def test_tensors_of_another_device():
    from b2lstm import operators
    assert b2lstm.lib().b2_current_device() >= -1
    ops, library = operators._ops(), b2lstm.lib()
    real = {name: C.cast(getattr(library, name), C.c_void_p).value for name in operators._BOUND}
    current = C.CFUNCTYPE(C.c_int)(lambda: 1)                     # as if device 1 was the current one
    on = lambda d, *s, **k: FakeOn(d, *s, **k)  # noqa: E731
    i32, ws = dict(dtype="torch.int32"), dict(dtype="torch.uint8")
    try:
        ops.bind(dict(real, b2_current_device=C.cast(current, C.c_void_p).value), b2lstm.B2Error)
        refused("out is on device 0, the current one is 1", b2lstm.embedding_forward, on(0, 4, 8), on(1, 10, 8), on(1, 4, **i32))
        refused("table is on device 2", b2lstm.embedding_forward, on(1, 4, 8), on(2, 10, 8), on(1, 4, **i32))
        refused("tokens is on device 0", b2lstm.embedding_forward, on(1, 4, 8), on(1, 10, 8), on(0, 4, **i32))
        refused("workspace is on device 0", b2lstm.embedding_backward, on(1, 10, 8), on(1, 4, 8), on(1, 4, **i32), workspace=on(0, 1 << 20, **ws))
        refused("not on the GPU", b2lstm.embedding_forward, on(-1, 4, 8), on(1, 10, 8), on(1, 4, **i32))
        refused("lse is on device 0", b2lstm.logprob_forward, on(1, 4, 8), on(1, 4, **i32), on(1, 4), on(0, 4))
        refused("mask is on device 0", b2lstm.logprob_forward, on(1, 4, 8), on(1, 4, **i32), on(1, 4), on(1, 4), mask=on(0, 8, dtype="torch.bool"))
        refused("h is on device 0", b2lstm.block_norm_forward, on(1, 4, 16), None, None, on(0, 4, 16))
        refused("devices .0, 1.", b2lstm.TensorList, [on(0, 3), on(1, 3)])
        refused("devices .0, 1.", b2lstm.TensorList, [on(1, 3)], [on(0, 3, address=8192)])
        refused("tensors are on device 0, the current one is 1", b2lstm.gradient_norm, b2lstm.TensorList([on(0, 3)]), on(1, 1), workspace=on(1, 1 << 16, **ws))
        refused("norm is on device 0", b2lstm.gradient_clip, b2lstm.TensorList([on(1, 3)]), 1.0, on(0, 1), workspace=on(1, 1 << 16, **ws))
        # on the current device the calls go on, to the next thing that is wrong
        refused("error -5.*aligned", b2lstm.embedding_forward, on(1, 4, 8), on(1, 10, 8, address=4098), on(1, 4, **i32))
        refused("error -1.*needed", b2lstm.gradient_clip, b2lstm.TensorList([on(1, 3)]), 1.0, on(1, 1), workspace=on(1, 8, **ws))
        # one that does not say where it is, is taken at its word
        refused("error -5.*aligned", b2lstm.embedding_forward, Fake(4, 8), Fake(10, 8, address=4098), TOK)
    finally:
        ops.bind(real, b2lstm.B2Error)


def test_a_norm_gradient_in_place_of_a_gate_for_several_frames():
    """other frames still read the gate's rows: refused, and accepted where every frame has its own"""
    x, o, st, ws = Fake(4, 16), Fake(4, 16, address=8192), Fake(4, 4, address=16384), dict(workspace=Fake(1 << 24, dtype="torch.uint8"))
    gate = Fake(2, 16, address=1 << 20)
    for at in (0, 1):
        outs = [Fake(4, 16, address=1 << 21), Fake(4, 16, address=1 << 22)]
        outs[at] = Fake(4, 16, address=1 << 20)
        refused("error -5.*place of the gate", b2lstm.block_norm_backward, *outs, x, None, None, o, st, gate=gate, **ws)
        refused("error -5.*place of the gate", b2lstm.block_norm_backward, *outs, x, None, None, o, st, gate=Fake(4, 16, address=1 << 20, stride=(24, 1)), **ws)

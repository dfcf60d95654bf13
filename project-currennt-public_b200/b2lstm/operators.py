"""The operators of a token model around the recurrent layers (include/b2lstm.h: b2_embedding_*, b2_block_norm_*, b2_logprob_*,
b2_gradient_*), on tensors: any object with data_ptr(), shape, stride(), dtype and is_cuda, e.g. torch CUDA tensors.

Shapes, element types and leading dimensions come from the tensors and are checked here; the library checks the rest.  Rows may lie
apart (a slice of a wider tensor), channels have to be contiguous.  Outputs are the caller's tensors.  `stream` is a raw stream handle
(None: the default stream); `workspace` a uint8 tensor of at least as many bytes as the matching _workspace function tells.
"""
import ctypes as C

from .lib import B2Error, _check, lib

_CODES = {"float32": 0, "bfloat16": 1, "float16": 2}
_F32, _I32, _BYTES = ("float32",), ("int32",), ("uint8", "int8", "bool")
_names = {}     # the name of a dtype, looked up once


def _name(dtype):
    name = _names.get(dtype)
    if name is None:
        name = _names[dtype] = str(dtype).split(".")[-1]
    return name


def _type(t):
    """element type code of a tensor"""
    code = _CODES.get(_names.get(t.dtype) or _name(t.dtype))
    if code is None:
        raise B2Error("element type %s (float32, bfloat16 or float16)" % t.dtype)
    return code


def _rows(t, name, rows=None, cols=None, like=None):
    """(address, leading dimension) of a matrix; (None, 0) for None"""
    if t is None:
        return None, 0
    shape = t.shape
    if len(shape) != 2 or (rows is not None and shape[0] != rows) or (cols is not None and shape[1] != cols):
        raise B2Error("%s has the shape %s, not (%s, %s)" % (name, tuple(shape), "rows" if rows is None else rows, "columns" if cols is None else cols))
    if not t.is_cuda:
        raise B2Error("%s is not on the GPU" % name)
    if like is not None and t.dtype != like:
        raise B2Error("%s has the element type %s, not %s" % (name, t.dtype, like))
    n, width = shape
    ld, unit = t.stride()
    if (unit != 1 and width > 1) or (ld < width and n > 1):
        raise B2Error("%s has the strides (%d, %d): its rows have to be contiguous and apart" % (name, ld, unit))
    return t.data_ptr(), ld if ld > width else width


def _vector(t, name, n, dtype):
    """address of a contiguous tensor of n elements; None for None"""
    if t is None:
        return None
    if not t.is_cuda:
        raise B2Error("%s is not on the GPU" % name)
    if (_names.get(t.dtype) or _name(t.dtype)) not in dtype:
        raise B2Error("%s has the element type %s, not %s" % (name, t.dtype, " or ".join(dtype)))
    if t.numel() != n or not t.is_contiguous():
        raise B2Error("%s has the shape %s and strides %s, not %d contiguous elements" % (name, tuple(t.shape), tuple(t.stride()), n))
    return t.data_ptr()


def _workspace(t):
    if t is None:
        return None, 0
    if not t.is_cuda or not t.is_contiguous():
        raise B2Error("the workspace is not a contiguous tensor on the GPU")
    return t.data_ptr(), t.numel() * t.element_size()


def embedding_forward(out, table, tokens, scale=1.0, stream=None):
    """out[r] = scale * table[tokens[r]]: tokens int32 [n], table [vocab, dim], out [n, dim]; zeros for a negative token"""
    n = tokens.numel()
    vocab, dim = table.shape
    o, ld_o = _rows(out, "out", n, dim)
    w, ld_w = _rows(table, "table")
    _check(lib().b2_embedding_forward(o, _type(out), ld_o, w, _type(table), ld_w, vocab, dim, _vector(tokens, "tokens", n, _I32), n, scale, stream))


def embedding_backward_workspace(n, vocab, dim):
    return int(lib().b2_embedding_backward_workspace(n, vocab, dim))


def embedding_backward(dtable, dout, tokens, scale=1.0, accumulate=False, workspace=None, stream=None):
    """dtable[v] = scale * sum of dout[r] over the rows with tokens[r] = v (added to dtable with accumulate)"""
    n = tokens.numel()
    vocab, dim = dtable.shape
    d, ld_d = _rows(dtable, "dtable")
    g, ld_g = _rows(dout, "dout", n, dim)
    ws, size = _workspace(workspace)
    _check(lib().b2_embedding_backward(d, _type(dtable), ld_d, vocab, dim, g, _type(dout), ld_g, _vector(tokens, "tokens", n, _I32), n, scale,
                                       int(accumulate), ws, size, stream))


class _BlockNorm(C.Structure):
    _fields_ = [("type", C.c_int), ("dim", C.c_int), ("rows", C.c_longlong), ("layer_norm", C.c_int), ("eps", C.c_float),
                ("residual_scale", C.c_float), ("pat_types", C.c_void_p), ("w_pre", C.c_void_p), ("b_pre", C.c_void_p), ("w_post", C.c_void_p),
                ("b_post", C.c_void_p), ("gate", C.c_void_p), ("gate_rows", C.c_longlong), ("ld_gate", C.c_longlong), ("stats", C.c_void_p)]


def _block_norm(like, w_pre, b_pre, w_post, b_post, gate, stats, pat_types, layer_norm, eps, residual_scale):
    rows, dim = like.shape
    g, ld_g = _rows(gate, "gate", None, dim, like.dtype)
    return _BlockNorm(_type(like), dim, rows, int(layer_norm), eps, residual_scale, _vector(pat_types, "pat_types", rows, _BYTES),
                      _vector(w_pre, "w_pre", dim, _F32), _vector(b_pre, "b_pre", dim, _F32), _vector(w_post, "w_post", dim, _F32),
                      _vector(b_post, "b_post", dim, _F32), g, gate.shape[0] if gate is not None else 0, ld_g,
                      _vector(stats, "stats", 4 * rows, _F32))


def block_norm_forward(x, f, y, h, w_pre=None, b_pre=None, w_post=None, b_post=None, gate=None, stats=None, pat_types=None, layer_norm=False,
                       eps=1e-5, residual_scale=1.0, stream=None):
    """y = x + residual_scale * gate * (w_post * norm(f) + b_post) and h = w_pre * norm(y) + b_pre over [rows, dim] tensors; f None: y = x
    (y may be None); h None: no norm behind the last block.  stats float32 [rows, 4] for the backward pass."""
    d = _block_norm(x, w_pre, b_pre, w_post, b_post, gate, stats, pat_types, layer_norm, eps, residual_scale)
    args = []
    for t, name in ((x, "x"), (f, "f"), (y, "y"), (h, "h")):
        args += _rows(t, name, d.rows, d.dim, x.dtype)
    _check(lib().b2_block_norm_forward(C.byref(d), *args, stream))


def block_norm_backward_workspace(rows, dim, gate_rows=0):
    return int(lib().b2_block_norm_backward_workspace(rows, dim, gate_rows))


def block_norm_backward(dx, df, dy, dh, y, f, stats, w_pre=None, w_post=None, b_post=None, gate=None, dgate=None, dw_pre=None, db_pre=None,
                        dw_post=None, db_post=None, pat_types=None, layer_norm=False, residual_scale=1.0, workspace=None, stream=None):
    """The gradients of block_norm_forward from those of y (dy) and h (dh); outputs that are None are left out."""
    like = next((t for t in (dy, dh) if t is not None), None)
    if like is None:
        raise B2Error("dy or dh is needed")
    if dgate is not None and gate is None:
        raise B2Error("dgate is given without the gate")
    d = _block_norm(like, w_pre, None, w_post, b_post, gate, stats, pat_types, layer_norm, 0.0, residual_scale)
    args = []
    for t, name in ((dx, "dx"), (df, "df")):
        args += _rows(t, name, d.rows, d.dim, like.dtype)
    args += _rows(dgate, "dgate", d.gate_rows, d.dim, like.dtype)
    args += [_vector(t, name, d.dim, _F32) for t, name in ((dw_pre, "dw_pre"), (db_pre, "db_pre"), (dw_post, "dw_post"), (db_post, "db_post"))]
    for t, name in ((dy, "dy"), (dh, "dh"), (y, "y"), (f, "f")):
        args += _rows(t, name, d.rows, d.dim, like.dtype)
    _check(lib().b2_block_norm_backward(C.byref(d), *args, *_workspace(workspace), stream))


def _mask(mask, rows, vocab):
    """address and leading dimension of a [vocab] or [rows, vocab] tensor of bytes"""
    if mask is None:
        return None, 0
    if len(mask.shape) == 1:
        return _vector(mask, "mask", vocab, _BYTES), 0
    if _name(mask.dtype) not in _BYTES:
        raise B2Error("mask has the element type %s" % mask.dtype)
    return _rows(mask, "mask", rows, vocab)


def logprob_forward(logits, tokens, logprob, lse, entropy=None, top_tokens=None, top_logprobs=None, mask=None, scale=1.0, stream=None):
    """Log probabilities of tokens (int32 [rows]) under logits [rows, vocab]: logprob, lse, entropy float32 [rows], the most likely tokens in
    top_tokens int32 / top_logprobs float32 [rows, top].  mask: uint8 or bool [vocab] or [rows, vocab], 0 = not allowed."""
    rows, vocab = logits.shape
    x, ld = _rows(logits, "logits")
    m, ld_m = _mask(mask, rows, vocab)
    top = top_tokens.shape[-1] if top_tokens is not None else 0
    _check(lib().b2_logprob_forward(x, _type(logits), rows, vocab, ld, m, ld_m, scale, _vector(tokens, "tokens", rows, _I32),
                                    _vector(logprob, "logprob", rows, _F32), _vector(lse, "lse", rows, _F32), _vector(entropy, "entropy", rows, _F32),
                                    top, _vector(top_tokens, "top_tokens", rows * top, _I32), _vector(top_logprobs, "top_logprobs", rows * top, _F32),
                                    stream))


def logprob_backward(dlogits, logits, tokens, lse, dlogprob, entropy=None, dentropy=None, mask=None, scale=1.0, stream=None):
    """The gradient of sum(dlogprob * logprob + dentropy * entropy) with respect to the logits; dlogits may be logits."""
    rows, vocab = logits.shape
    d, ld_d = _rows(dlogits, "dlogits", rows, vocab, logits.dtype)
    x, ld = _rows(logits, "logits")
    m, ld_m = _mask(mask, rows, vocab)
    _check(lib().b2_logprob_backward(d, ld_d, x, _type(logits), rows, vocab, ld, m, ld_m, scale, _vector(tokens, "tokens", rows, _I32),
                                     _vector(lse, "lse", rows, _F32), _vector(dlogprob, "dlogprob", rows, _F32),
                                     _vector(entropy, "entropy", rows, _F32), _vector(dentropy, "dentropy", rows, _F32), stream))


class _Tensor(C.Structure):
    _fields_ = [("data", C.c_void_p), ("count", C.c_size_t), ("type", C.c_int)]


class TensorList:
    """The gradients of a model as one argument, built once: a list of contiguous tensors and, where they are not scaled in place, the
    tensors that take the scaled ones.  Holds references to them."""

    def __init__(self, tensors, out=None):
        self.tensors, self.out = list(tensors), None if out is None else list(out)
        self.n = len(self.tensors)
        if self.out is not None and len(self.out) != self.n:
            raise B2Error("%d tensors and %d outputs" % (self.n, len(self.out)))
        self._in, self._out = self._array(self.tensors), None if out is None else self._array(self.out)

    @staticmethod
    def _array(tensors):
        a = (_Tensor * len(tensors))()
        for i, t in enumerate(tensors):
            if not t.is_cuda or not t.is_contiguous():
                raise B2Error("tensor %d is not a contiguous tensor on the GPU" % i)
            a[i] = _Tensor(t.data_ptr(), t.numel(), _type(t))
        return a


def gradient_norm_workspace():
    return int(lib().b2_gradient_norm_workspace())


def gradient_norm(tensors, norm, workspace=None, stream=None):
    """norm (float32 [1]) = the L2 norm over all elements of a TensorList"""
    _check(lib().b2_gradient_norm(tensors._in, tensors.n, _vector(norm, "norm", 1, _F32), *_workspace(workspace), stream))


def gradient_clip(tensors, max_norm, norm, workspace=None, stream=None):
    """The same, and the tensors scaled by min(1, max_norm / norm), in place or into the list's outputs"""
    _check(lib().b2_gradient_clip(tensors._in, tensors._out, tensors.n, max_norm, _vector(norm, "norm", 1, _F32), *_workspace(workspace), stream))

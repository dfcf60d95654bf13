"""The operators of a token model around the recurrent layers (include/b2lstm.h: b2_embedding_*, b2_block_norm_*, b2_logprob_*,
b2_gradient_*, b2_distill_*, b2_beam_*, b2_int8_*), on tensors: any object with data_ptr(), shape, stride(), dtype and is_cuda, e.g. torch CUDA tensors.  Calls go to the current
CUDA device; tensors that say where they are (get_device()) are refused if that is another one.

Shapes, element types and leading dimensions come from the tensors and are checked on the way (csrc/binding.cpp); the library checks the rest.  Rows may lie
apart (a slice of a wider tensor), channels have to be contiguous.  Outputs are the caller's tensors.  `stream` is a raw stream handle,
None the legacy default stream, as everywhere in this package: under torch.cuda.stream(s) that is not the stream the tensors are made on, and the call is not
ordered with them unless it is given s.cuda_stream; `workspace` a uint8 tensor of at least as many bytes as the matching _workspace function tells.
"""
import ctypes as C

from .lib import B2Error, lib

try:
    from . import _tensors      # csrc/binding.cpp
except ImportError:             # not built: the first call says so
    _tensors = None

_BOUND = ("b2_last_error_string", "b2_current_device", "b2_embedding_forward", "b2_embedding_backward", "b2_block_norm_forward", "b2_block_norm_backward", "b2_logprob_forward",
          "b2_logprob_backward", "b2_gradient_norm", "b2_gradient_clip", "b2_distill_forward", "b2_distill_backward", "b2_beam_select", "b2_beam_reorder",
          "b2_int8_quantize", "b2_int8_product")
_ready = None


def _ops():
    """the binding, with the library's functions in it"""
    global _ready
    if _ready is None:
        if _tensors is None:
            raise B2Error("b2lstm/_tensors.so is not built (make -C csrc)")
        library = lib()
        _tensors.bind({name: C.cast(getattr(library, name), C.c_void_p).value for name in _BOUND}, B2Error)
        _ready = _tensors
    return _ready


def embedding_forward(out, table, tokens, scale=1.0, stream=None):
    """out[r] = scale * table[tokens[r]]: tokens int32 [n], table [vocab, dim], out [n, dim]; zeros for a negative token"""
    (_ready or _ops()).embedding_forward(out, table, tokens, scale, stream)


def embedding_backward_workspace(n, vocab, dim):
    return int(lib().b2_embedding_backward_workspace(n, vocab, dim))


def embedding_backward(dtable, dout, tokens, scale=1.0, accumulate=False, workspace=None, stream=None):
    """dtable[v] = scale * sum of dout[r] over the rows with tokens[r] = v (added to dtable with accumulate)"""
    (_ready or _ops()).embedding_backward(dtable, dout, tokens, scale, accumulate, workspace, stream)


def block_norm_forward(x, f, y, h, w_pre=None, b_pre=None, w_post=None, b_post=None, gate=None, stats=None, pat_types=None, layer_norm=False,
                       eps=1e-5, residual_scale=1.0, stream=None):
    """y = x + residual_scale * gate * (w_post * norm(f) + b_post) and h = w_pre * norm(y) + b_pre over [rows, dim] tensors; f None: y = x
    (y may be None); h None: no norm behind the last block.  stats float32 [rows, 4] for the backward pass."""
    (_ready or _ops()).block_norm_forward(x, f, y, h, w_pre, b_pre, w_post, b_post, gate, stats, pat_types, layer_norm, eps, residual_scale, stream)


def block_norm_backward_workspace(rows, dim, gate_rows=0):
    return int(lib().b2_block_norm_backward_workspace(rows, dim, gate_rows))


def block_norm_backward(dx, df, dy, dh, y, f, stats, w_pre=None, w_post=None, b_post=None, gate=None, dgate=None, dw_pre=None, db_pre=None,
                        dw_post=None, db_post=None, pat_types=None, layer_norm=False, residual_scale=1.0, workspace=None, stream=None):
    """The gradients of block_norm_forward from those of y (dy) and h (dh); outputs that are None are left out."""
    (_ready or _ops()).block_norm_backward(dx, df, dy, dh, y, f, dgate, dw_pre, db_pre, dw_post, db_post, w_pre, None, w_post, b_post, gate, stats, pat_types,
                                           layer_norm, 0.0, residual_scale, workspace, stream)


def logprob_forward(logits, tokens, logprob, lse, entropy=None, top_tokens=None, top_logprobs=None, mask=None, scale=1.0, stream=None):
    """Log probabilities of tokens (int32 [rows]) under logits [rows, vocab]: logprob, lse, entropy float32 [rows], the most likely tokens in
    top_tokens int32 / top_logprobs float32 [rows, top].  mask: uint8 or bool [vocab] or [rows, vocab], 0 = not allowed."""
    (_ready or _ops()).logprob_forward(logits, tokens, logprob, lse, entropy, top_tokens, top_logprobs, mask, scale, stream)


def logprob_backward(dlogits, logits, tokens, lse, dlogprob, entropy=None, dentropy=None, mask=None, scale=1.0, stream=None):
    """The gradient of sum(dlogprob * logprob + dentropy * entropy) with respect to the logits; dlogits may be logits."""
    (_ready or _ops()).logprob_backward(dlogits, logits, tokens, lse, dlogprob, entropy, dentropy, mask, scale, stream)


_CODES = {"float32": 0, "bfloat16": 1, "float16": 2}


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
        devices = {t.get_device() for t in self.tensors + (self.out or []) if hasattr(t, "get_device")}
        if len(devices) > 1:
            raise B2Error("the tensors are on the devices %s" % sorted(devices))
        self._device = devices.pop() if devices else -1
        self._at, self._out_at = C.addressof(self._in), 0 if out is None else C.addressof(self._out)

    @staticmethod
    def _array(tensors):
        a = (_Tensor * len(tensors))()
        for i, t in enumerate(tensors):
            if not t.is_cuda or not t.is_contiguous():
                raise B2Error("tensor %d is not a contiguous tensor on the GPU" % i)
            code = _CODES.get(str(t.dtype).split(".")[-1])
            if code is None:
                raise B2Error("tensor %d has the element type %s (float32, bfloat16 or float16)" % (i, t.dtype))
            a[i] = _Tensor(t.data_ptr(), t.numel(), code)
        return a


def gradient_norm_workspace():
    return int(lib().b2_gradient_norm_workspace())


def gradient_norm(tensors, norm, workspace=None, stream=None):
    """norm (float32 [1]) = the L2 norm over all elements of a TensorList"""
    (_ready or _ops()).gradient_norm(tensors._at, tensors.n, tensors._device, norm, workspace, stream)


def gradient_clip(tensors, max_norm, norm, workspace=None, stream=None):
    """The same, and the tensors scaled by min(1, max_norm / norm), in place or into the list's outputs"""
    (_ready or _ops()).gradient_clip(tensors._at, tensors._out_at, tensors.n, tensors._device, max_norm, norm, workspace, stream)


def distill_forward(logits, top_tokens, top_logprobs, loss, lse, lse_rest=None, scale=1.0, stream=None):
    """Divergence of the rows of logits [rows, vocab] from a teacher's most likely tokens: top_tokens int32 and top_logprobs float32 [rows, top] as
    logprob_forward leaves them, loss and lse float32 [rows].  With lse_rest (float32 [rows]) the rest of the vocabulary counts as one more outcome."""
    (_ready or _ops()).distill_forward(logits, top_tokens, top_logprobs, loss, lse, lse_rest, scale, stream)


def distill_backward(dlogits, logits, top_tokens, top_logprobs, lse, dloss, lse_rest=None, scale=1.0, accumulate=False, stream=None):
    """The gradient of sum(dloss * loss) with respect to the logits (added to dlogits with accumulate; dlogits may else be logits)"""
    (_ready or _ops()).distill_backward(dlogits, logits, top_tokens, top_logprobs, lse, lse_rest, dloss, scale, accumulate, stream)


def beam_select_workspace(groups, beams, vocab, top):
    return int(lib().b2_beam_select_workspace(groups, beams, vocab, top))


def beam_select(logits, scores, top_scores, top_beams, top_tokens, finished=None, weights=None, end_token=0, mask=None, scale=1.0, workspace=None,
                stream=None):
    """The best continuations of the beams of each sequence: logits [groups * beams, vocab], scores float32 [groups * beams], results [groups, top]
    (scores float32; the beam each one continues and its token int32).  finished uint8 or bool, weights float32 [groups * beams]; mask as for
    logprob_forward."""
    (_ready or _ops()).beam_select(logits, scores, top_scores, top_beams, top_tokens, finished, weights, end_token, mask, scale, workspace, stream)


class _State(C.Structure):
    _fields_ = [("data", C.c_void_p), ("out", C.c_void_p), ("outer", C.c_longlong), ("row_bytes", C.c_longlong)]


class StateList:
    """What the beams of a search carry along, as one argument, built once: contiguous tensors of any element types, the axis of each that runs over
    the beams of all sequences (an int for all, or one for each), and, where they are not reordered in place, the tensors that take the
    reordered ones.  Holds references to them."""

    def __init__(self, tensors, axes=0, out=None):
        self.tensors, self.out = list(tensors), None if out is None else list(out)
        self.n = len(self.tensors)
        axes = [axes] * self.n if isinstance(axes, int) else list(axes)
        if len(axes) != self.n or (self.out is not None and len(self.out) != self.n):
            raise B2Error("%d tensors, %d axes and %s outputs" % (self.n, len(axes), "no" if out is None else len(self.out)))
        self._in, rows = (_State * self.n)(), set()
        for i, t in enumerate(self.tensors):
            to = t if self.out is None else self.out[i]
            shape = tuple(t.shape)
            for x in (t, to):
                if not x.is_cuda or not x.is_contiguous():
                    raise B2Error("tensor %d is not a contiguous tensor on the GPU" % i)
            if tuple(to.shape) != shape or to.dtype != t.dtype:
                raise B2Error("output %d has the shape %s and the element type %s, not %s and %s" % (i, tuple(to.shape), to.dtype, shape, t.dtype))
            if not 0 <= axes[i] < len(shape):
                raise B2Error("tensor %d has the shape %s: no axis %d" % (i, shape, axes[i]))
            outer, inner = 1, t.element_size()
            for n in shape[:axes[i]]:
                outer *= n
            for n in shape[axes[i] + 1:]:
                inner *= n
            rows.add(shape[axes[i]])
            self._in[i] = _State(t.data_ptr(), to.data_ptr(), outer, inner)
        if len(rows) > 1:
            raise B2Error("the tensors have %s beams" % sorted(rows))
        devices = {t.get_device() for t in self.tensors + (self.out or []) if hasattr(t, "get_device")}
        if len(devices) > 1:
            raise B2Error("the tensors are on the devices %s" % sorted(devices))
        self.rows = rows.pop() if rows else -1
        self._device = devices.pop() if devices else -1
        self._at = C.addressof(self._in)


def beam_reorder(states, parents, stream=None):
    """The tensors of a StateList by parents (int32 [groups, beams]): row g * beams + b becomes row g * beams + parents[g, b], zeros for a parent that is
    no beam"""
    (_ready or _ops()).beam_reorder(states._at, states.n, states._device, states.rows, parents, stream)


def int8_quantize(q, scales, x, stream=None):
    """q (int8) = x over scales, scales (float32 [rows]) = the largest magnitudes of the rows of x over 127.  int8_product wants rows of int8 that start at
    multiples of 16 bytes: torch.empty(rows, (dim + 15) // 16 * 16, dtype=torch.int8)[:, :dim]"""
    (_ready or _ops()).int8_quantize(q, scales, x, stream)


def int8_product_workspace(rows, channels, dim):
    return int(lib().b2_int8_product_workspace(rows, channels, dim))


def int8_product(out, x, w, w_scales, bias=None, x_scales=None, workspace=None, stream=None):
    """out [rows, channels] = x [rows, dim] times w [channels, dim] (int8, w_scales float32 [channels]) in 8-bit integers, plus bias (float32 [channels]); x is
    quantised in the call (with a workspace), or int8 with its x_scales (float32 [rows])"""
    (_ready or _ops()).int8_product(out, x, x_scales, w, w_scales, bias, workspace, stream)

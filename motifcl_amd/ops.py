"""Thin Python front of the C ABI.  torch is used only as the owner of device
memory and of the current HIP stream; every computation happens in
libmotifcl_amd.so."""
import collections
import ctypes

import torch

from . import lib as _lib


def _stream():
    return torch.cuda.current_stream().cuda_stream or None


def _buf(t, dtype):
    if not t.is_cuda:
        raise ValueError("expected a device tensor")
    if t.dtype != dtype:
        raise ValueError("expected dtype %s, got %s" % (dtype, t.dtype))
    if not t.is_contiguous():
        raise ValueError("expected a contiguous tensor")
    return t.data_ptr(), t.numel() * t.element_size()


def apply_update_dense(state, scale, v, grad_w, C, lr, lr_scale, rms_beta, rms_eps, seed,
                       in_features=None, out_features=None):
    """In-place update-only step (CounterStateLinear::apply_update_seed)."""
    L = _lib.load()
    if in_features is None:
        out_features, in_features = grad_w.shape
    _lib.check(L.mcc_compact_counter_apply_update_dense(
        _stream(), *_buf(state, torch.uint8), *_buf(scale, torch.float32), *_buf(v, torch.float32),
        *_buf(grad_w, torch.float32), C, in_features, out_features,
        lr, lr_scale, rms_beta, rms_eps, seed & 0xFFFFFFFF))


class UpdateBatch:
    """A reusable descriptor list for apply_update_dense_batched: tensors are
    (state, scale, v, grad_w) device tensors with grad_w of shape [out, in]."""

    def __init__(self, tensors, lr, seeds):
        self._keep = list(tensors)
        n = len(self._keep)
        self.array = (_lib.CounterTensor * n)()
        for i, (state, scale, v, grad_w) in enumerate(self._keep):
            out_features, in_features = grad_w.shape
            d = self.array[i]
            d.state, d.state_nbytes = _buf(state, torch.uint8)
            d.scale, d.scale_nbytes = _buf(scale, torch.float32)
            d.v, d.v_nbytes = _buf(v, torch.float32)
            d.grad_w, d.grad_w_nbytes = _buf(grad_w, torch.float32)
            d.in_features, d.out_features = in_features, out_features
            d.lr = lr[i] if isinstance(lr, (list, tuple)) else lr
            d.seed = seeds[i] & 0xFFFFFFFF
        self.n = n

    def set_seeds(self, seeds):
        for i in range(self.n):
            self.array[i].seed = seeds[i] & 0xFFFFFFFF


def apply_update_dense_batched(batch, C, lr_scale, rms_beta, rms_eps):
    """In-place update-only step of every tensor of an UpdateBatch, one call."""
    L = _lib.load()
    _lib.check(L.mcc_compact_counter_apply_update_dense_batched(
        _stream(), batch.array, batch.n, C, lr_scale, rms_beta, rms_eps))


class FusedBatch:
    """A reusable descriptor list for apply_update_fused_batched: tensors are
    (state, scale, v, grad_out [batch, out], x [batch, in]) device tensors."""

    def __init__(self, tensors, lr, seeds):
        self._keep = list(tensors)
        n = len(self._keep)
        self.array = (_lib.FusedTensor * n)()
        for i, (state, scale, v, grad_out, x) in enumerate(self._keep):
            batch, out_features = grad_out.shape
            d = self.array[i]
            d.state, d.state_nbytes = _buf(state, torch.uint8)
            d.scale, d.scale_nbytes = _buf(scale, torch.float32)
            d.v, d.v_nbytes = _buf(v, torch.float32)
            d.grad_out, d.grad_out_nbytes = _buf(grad_out, torch.float32)
            d.x, d.x_nbytes = _buf(x, torch.float32)
            d.in_features, d.out_features, d.batch = x.shape[1], out_features, batch
            d.lr = lr[i] if isinstance(lr, (list, tuple)) else lr
            d.seed = seeds[i] & 0xFFFFFFFF
        self.n = n

    def set_seeds(self, seeds):
        for i in range(self.n):
            self.array[i].seed = seeds[i] & 0xFFFFFFFF

    def workspace_nbytes(self):
        return int(_lib.load().mcc_compact_counter_fused_batched_workspace_nbytes(self.array, self.n))


def apply_update_fused_batched(batch, workspace, C, lr_scale, rms_beta, rms_eps):
    """In-place fused step of every tensor of a FusedBatch in a handful of launches."""
    L = _lib.load()
    _lib.check(L.mcc_compact_counter_apply_update_fused_batched(
        _stream(), batch.array, batch.n, *_buf(workspace, torch.uint8), C, lr_scale, rms_beta, rms_eps))


def fused_workspace_nbytes(in_features, out_features, batch):
    return int(_lib.load().mcc_compact_counter_fused_workspace_nbytes(in_features, out_features, batch))


def fused_strip_workspace_nbytes(in_features, out_features, batch):
    """Size of the small workspace of the accumulator-resident fused step; 0 if unsupported."""
    return int(_lib.load().mcc_compact_counter_fused_strip_workspace_nbytes(in_features, out_features, batch))


def fused_check(workspace, in_features, out_features, batch):
    """Waits for the stream and raises MccError if a strip-workspace step gave up a wait."""
    L = _lib.load()
    ptr, nbytes = (0, 0) if workspace is None else (workspace.data_ptr(), workspace.numel() * workspace.element_size())
    _lib.check(L.mcc_compact_counter_fused_check(_stream(), ptr, nbytes, in_features, out_features, batch))


def apply_update_fused(state, scale, v, grad_out, x, workspace, C, lr, lr_scale, rms_beta, rms_eps,
                       seed):
    """In-place fused step (CounterStateLinear::apply_update_backward)."""
    L = _lib.load()
    batch, out_features = grad_out.shape
    in_features = x.shape[1]
    if x.shape[0] != batch:
        raise ValueError("x and grad_out disagree on the batch size")
    _lib.check(L.mcc_compact_counter_apply_update_fused(
        _stream(), *_buf(state, torch.uint8), *_buf(scale, torch.float32), *_buf(v, torch.float32),
        *_buf(grad_out, torch.float32), *_buf(x, torch.float32),
        workspace.data_ptr(), workspace.numel() * workspace.element_size(),
        C, in_features, out_features, batch, lr, lr_scale, rms_beta, rms_eps, seed & 0xFFFFFFFF))


NOALLOC_WORKSPACE_NBYTES = 32 << 20  # MCC_NOALLOC_WORKSPACE_NBYTES of include/motifcl_amd.h


def apply_update_fused_static(state, scale, v, grad_out, x, C, lr, lr_scale, rms_beta, rms_eps, seed):
    """The fused step on the library's own static workspace: the call allocates nothing."""
    L = _lib.load()
    batch, out_features = grad_out.shape
    in_features = x.shape[1]
    if x.shape[0] != batch:
        raise ValueError("x and grad_out disagree on the batch size")
    _lib.check(L.mcc_compact_counter_apply_update_fused_static(
        _stream(), *_buf(state, torch.uint8), *_buf(scale, torch.float32), *_buf(v, torch.float32),
        *_buf(grad_out, torch.float32), *_buf(x, torch.float32),
        C, in_features, out_features, batch, lr, lr_scale, rms_beta, rms_eps, seed & 0xFFFFFFFF))


def matmul_transpose_a(a, b, out=None):
    """c[m,n] = a[k,m]^T . b[k,n]."""
    L = _lib.load()
    k, m = a.shape
    k2, n = b.shape
    if k != k2:
        raise ValueError("matmul_transpose_a: leading dimensions differ")
    if out is None:
        out = torch.empty((m, n), dtype=torch.float32, device=a.device)
    _lib.check(L.mcc_matmul_transpose_a_f32(_stream(), *_buf(a, torch.float32), *_buf(b, torch.float32),
                                            *_buf(out, torch.float32), k, m, n))
    return out


def decode_weight(state, scale, C, in_features, out_features, out=None):
    L = _lib.load()
    w = out if out is not None else torch.empty((out_features, in_features), dtype=torch.float32, device=state.device)
    _lib.check(L.mcc_compact_counter_decode_weight(
        _stream(), *_buf(state, torch.uint8), *_buf(scale, torch.float32), *_buf(w, torch.float32),
        in_features, out_features, C))
    return w


def forward(x, state, scale, C, out_features, out=None):
    L = _lib.load()
    batch, in_features = x.shape
    y = out if out is not None else torch.empty((batch, out_features), dtype=torch.float32, device=x.device)
    _lib.check(L.mcc_compact_counter_forward_u8(
        _stream(), *_buf(x, torch.float32), *_buf(state, torch.uint8), *_buf(scale, torch.float32),
        *_buf(y, torch.float32), batch, in_features, out_features, C))
    return y


def backward_input(grad_out, state, scale, C, in_features, out=None):
    L = _lib.load()
    batch, out_features = grad_out.shape
    gx = out if out is not None else torch.empty((batch, in_features), dtype=torch.float32, device=grad_out.device)
    _lib.check(L.mcc_compact_counter_backward_input_u8(
        _stream(), *_buf(state, torch.uint8), *_buf(scale, torch.float32),
        *_buf(grad_out, torch.float32), *_buf(gx, torch.float32),
        batch, in_features, out_features, C))
    return gx


def sgd_update(param, grad, lr):
    """param -= lr * grad in place (sgd_update of MotifCL)."""
    L = _lib.load()
    _lib.check(L.mcc_sgd_update_f32(_stream(), *_buf(param, torch.float32), *_buf(grad, torch.float32),
                                    param.numel(), lr))


def adam_update(param, grad, m, v, lr, beta1, beta2, eps, step, weight_decay=0.0):
    """In-place Adam step with decoupled weight decay (adam_update_fast of MotifCL)."""
    L = _lib.load()
    _lib.check(L.mcc_adam_update_f32(_stream(), *_buf(param, torch.float32), *_buf(grad, torch.float32),
                                     *_buf(m, torch.float32), *_buf(v, torch.float32), param.numel(),
                                     lr, beta1, beta2, eps, step, weight_decay))


# ---- row-wise operators around the counter layers ------------------------------------------------
_ELEMENTS = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}  # MCC_ELEMENT_* of include/motifcl_amd.h
MOST_TOP = 128  # MCC_MOST_TOP

TokenLogProbs = collections.namedtuple("TokenLogProbs", "log_prob entropy lse top_ids top_log_probs")


def _rows(t, name):
    """(pointer, bytes, row stride), rows, row length and element type of a tensor whose last dimension is the
    row: contiguous, or two-dimensional with contiguous rows."""
    if not t.is_cuda:
        raise ValueError("expected a device tensor")
    element = _ELEMENTS.get(t.dtype)
    if element is None:
        raise ValueError("%s: expected float32, float16 or bfloat16, got %s" % (name, t.dtype))
    dims = t.dim()
    if dims == 0:
        raise ValueError("%s: expected at least one dimension" % name)
    shape = t.shape
    cols = stride = shape[-1]
    rows = shape[0] if dims == 2 else t.numel() // cols if cols else 0
    if not t.is_contiguous():
        if dims != 2 or (t.stride(1) != 1 and cols != 1):
            raise ValueError("%s: expected a contiguous tensor or a matrix with contiguous rows" % name)
        stride = t.stride(0)
    nbytes = ((rows - 1) * stride + cols) * (2 if element else 4) if rows else 0
    return (t.data_ptr(), nbytes, stride), rows, cols, element


def _same_rows(t, like, name):
    """(pointer, bytes, row stride) of a tensor with the shape, type and device of `like`."""
    if t.shape != like.shape or t.dtype != like.dtype or t.device != like.device:
        raise ValueError("%s: expected shape %s, %s on %s" % (name, tuple(like.shape), like.dtype, like.device))
    return _rows(t, name)[0]


def _out_rows(out, like, buf):
    """An output with the shape, type and device of `like`, whose _rows() gave `buf`: the caller's tensor or a new
    one; and its (pointer, bytes, row stride)."""
    if out is not None:
        return out, _same_rows(out, like, "out")
    if not like.is_contiguous():
        out = like.new_empty(like.shape)
        return out, _rows(out, "out")[0]
    out = torch.empty_like(like)
    return out, (out.data_ptr(), buf[1], buf[2])


def _numbers(t, dtype, shape, like, name):
    """(pointer, bytes) of a contiguous tensor of 4-byte numbers on the device of `like`; None gives a null pointer."""
    if t is None:
        return None, 0
    if t.shape != shape or t.device != like.device:
        raise ValueError("%s: expected shape %s on %s, got %s on %s" % (name, tuple(shape), like.device, tuple(t.shape),
                                                                       t.device))
    if t.dtype != dtype:
        raise ValueError("expected dtype %s, got %s" % (dtype, t.dtype))
    if not t.is_contiguous():
        raise ValueError("expected a contiguous tensor")
    return t.data_ptr(), 4 * t.numel()


def _new(like, shape, dtype=torch.float32):
    return like.new_empty(shape, dtype=dtype)


# The current stream's handle without a Stream object around it, a tenth of the time; torch's own code
# generators launch through it.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(fn, like, *args):
    """One call on the current stream of the device that `like` is on."""
    index = like.get_device()
    if index == torch.cuda.current_device():
        rc = fn(_raw_stream(index) or None, *args)
    else:
        with torch.cuda.device(index):
            rc = fn(_raw_stream(index) or None, *args)
    if rc != 0:
        _lib.check(rc)


def _lent(nbytes, workspace, like):
    """(pointer, bytes) and owner of a workspace: the caller's, or a new one (None if none is needed)."""
    if workspace is None:
        if nbytes == 0:
            return (None, 0), None
        workspace = _new(like, nbytes, torch.uint8)
        return (workspace.data_ptr(), nbytes), workspace
    if workspace.device != like.device:
        raise ValueError("workspace: expected a tensor on %s" % like.device)
    return _buf(workspace, torch.uint8), workspace


def layer_norm(x, gain=None, bias=None, eps=1e-5, out=None):
    """Layer norm of the rows (last dimension) of x: (y, mean, rstd).  gain and bias are float32 vectors;
    `out` may be x."""
    buf, rows, cols, element = _rows(x, "x")
    y, y_buf = _out_rows(out, x, buf)
    shape = x.shape[:-1]
    mean = _new(x, shape)
    rstd = torch.empty_like(mean)
    _call(_lib.load().mcc_layer_norm, x, *buf, *_numbers(gain, torch.float32, (cols,), x, "gain"),
          *_numbers(bias, torch.float32, (cols,), x, "bias"), *y_buf,
          mean.data_ptr(), 4 * rows, rstd.data_ptr(), 4 * rows, rows, cols, element, eps)
    return y, mean, rstd


def layer_norm_backward_workspace_nbytes(rows, cols, dtype):
    return int(_lib.load().mcc_layer_norm_backward_workspace_nbytes(rows, cols, _ELEMENTS[dtype]))


def layer_norm_backward(grad_out, x, mean, rstd, gain=None, bias=True, input_grad=True, out=None, workspace=None):
    """Gradients of layer_norm: (grad_x, grad_gain, grad_bias).  grad_gain is None without a gain, grad_bias with
    bias=False, grad_x with input_grad=False; `out` takes grad_x and may be grad_out or x."""
    L = _lib.load()
    buf, rows, cols, element = _rows(x, "x")
    grad_buf = _same_rows(grad_out, x, "grad_out")
    grad_x, x_out = _out_rows(out, x, buf) if input_grad else (None, (None, 0, 0))
    grad_gain = torch.empty_like(gain) if gain is not None else None
    grad_bias = _new(x, cols) if bias else None
    shape, n = x.shape[:-1], 4 * cols
    need = 0 if grad_gain is None and grad_bias is None else L.mcc_layer_norm_backward_workspace_nbytes(rows, cols, element)
    lent, workspace = _lent(need, workspace, x)
    _call(L.mcc_layer_norm_backward, x, *grad_buf, *buf, *_numbers(mean, torch.float32, shape, x, "mean"),
          *_numbers(rstd, torch.float32, shape, x, "rstd"), *_numbers(gain, torch.float32, (cols,), x, "gain"), *x_out,
          None if grad_gain is None else grad_gain.data_ptr(), n, None if grad_bias is None else grad_bias.data_ptr(), n,
          *lent, rows, cols, element)
    return grad_x, grad_gain, grad_bias


def token_log_probs_workspace_nbytes(rows, vocab, top, dtype):
    return int(_lib.load().mcc_token_log_probs_workspace_nbytes(rows, vocab, top, _ELEMENTS[dtype]))


def token_log_probs(logits, tokens=None, top=0, temperature=1.0, workspace=None):
    """TokenLogProbs of softmax(logits / temperature) along the last dimension: the log probability of `tokens`
    (int32, one a row; outside the vocabulary: 0; None without tokens), the entropy, the log of the sum of
    exponentials, and the `top` likeliest tokens with their log probabilities (None without)."""
    L = _lib.load()
    buf, rows, vocab, element = _rows(logits, "logits")
    shape = logits.shape[:-1]
    token_buf = _numbers(tokens, torch.int32, shape, logits, "tokens")
    entropy = _new(logits, shape)
    lse = torch.empty_like(entropy)
    log_prob = torch.empty_like(entropy) if tokens is not None else None
    ids = best = None
    if 0 < top <= MOST_TOP:
        ids, best = _new(logits, (*shape, top), torch.int32), _new(logits, (*shape, top))
    lent, workspace = _lent(L.mcc_token_log_probs_workspace_nbytes(rows, vocab, top, element) if top >= 0 else 0,
                            workspace, logits)
    n = 4 * rows
    _call(L.mcc_token_log_probs, logits, *buf, *token_buf,
          None if log_prob is None else log_prob.data_ptr(), n, entropy.data_ptr(), n, lse.data_ptr(), n,
          None if ids is None else ids.data_ptr(), n * top, None if best is None else best.data_ptr(), n * top,
          *lent, rows, vocab, top, element, temperature)
    return TokenLogProbs(log_prob, entropy, lse, ids, best)


def token_log_probs_backward(logits, tokens, lse, entropy, grad_log_prob, grad_entropy=None, temperature=1.0, out=None):
    """Gradient of the logits from the gradients of token_log_probs' log_prob and entropy (either may be None);
    lse and entropy are its results.  `out` may be logits."""
    buf, rows, vocab, element = _rows(logits, "logits")
    grad, grad_buf = _out_rows(out, logits, buf)
    shape = logits.shape[:-1]
    f32 = torch.float32
    _call(_lib.load().mcc_token_log_probs_backward, logits, *buf, *_numbers(tokens, torch.int32, shape, logits, "tokens"),
          *_numbers(lse, f32, shape, logits, "lse"), *_numbers(entropy, f32, shape, logits, "entropy"),
          *_numbers(grad_log_prob, f32, shape, logits, "grad_log_prob"),
          *_numbers(grad_entropy, f32, shape, logits, "grad_entropy"), *grad_buf,
          rows, vocab, element, temperature)
    return grad


def distill_top(logits, teacher_ids, teacher_logits, temperature=1.0, weight=None, grad=True, out=None):
    """Distillation from a teacher's top logits: (loss, grad_logits).  loss is temperature^2 * KL(teacher || student)
    of each row, grad_logits the gradient of sum(weight * loss) (None with grad=False).  teacher_ids (int32, an id
    outside the vocabulary is no entry) and teacher_logits (float32) hold the same number of entries a row, at most
    128; `out` takes grad_logits and may be logits."""
    buf, rows, vocab, element = _rows(logits, "logits")
    shape = logits.shape[:-1]
    if teacher_ids.dim() == 0:
        raise ValueError("teacher_ids: expected [..., entries]")
    top = teacher_ids.shape[-1]
    loss = _new(logits, shape)
    grad_logits, grad_buf = _out_rows(out, logits, buf) if grad else (None, (None, 0, 0))
    _call(_lib.load().mcc_distill_top, logits, *buf, *_numbers(teacher_ids, torch.int32, (*shape, top), logits, "teacher_ids"),
          *_numbers(teacher_logits, torch.float32, (*shape, top), logits, "teacher_logits"),
          *_numbers(weight, torch.float32, shape, logits, "weight"), loss.data_ptr(), 4 * rows, *grad_buf,
          rows, vocab, top, element, temperature)
    return loss, grad_logits


CONTRACTION_FP32, CONTRACTION_BF16X6 = 0, 1


def set_contraction_mode(mode):
    """Process-wide choice of the weight-gradient contraction: fp32 matrix instruction or split bf16."""
    _lib.check(_lib.load().mcc_set_contraction_mode(int(mode)))


def get_contraction_mode():
    return int(_lib.load().mcc_get_contraction_mode())


def fill_normal(t, stream_id, sigma):
    """t[i] = sigma * z_i from the library's counter-based generator (lowbias32 -> Box-Muller)."""
    ptr, nbytes = _buf(t, torch.float32)
    _lib.check(_lib.load().mcc_fill_normal_f32(_stream(), ptr, nbytes // 4, stream_id & 0xFFFFFFFF, sigma))
    return t


def fill_counter_state(state, stream_id, n_codes):
    """Packed state with every code uniform on [0, n_codes), same generator."""
    ptr, nbytes = _buf(state, torch.uint8)
    if nbytes % 3:
        raise ValueError("a packed state holds 3 bytes per group")
    _lib.check(_lib.load().mcc_fill_counter_state_u8(_stream(), ptr, nbytes // 3, stream_id & 0xFFFFFFFF, n_codes))
    return state


class ClockProbe:
    """Shader clock while other kernels run: a one-wave kernel on a side stream sleeps for
    `seconds` of the constant-rate wall clock and counts shader cycles over the same stretch.

        probe = ClockProbe(0.05)      # starts now, on its own stream
        ... launch the kernels under test on the current stream ...
        torch.cuda.synchronize()
        mhz = probe.mhz()
    """

    def __init__(self, seconds):
        L = _lib.load()
        khz = ctypes.c_int(0)
        _lib.check(L.mcc_wall_clock_khz(ctypes.byref(khz)))
        self._khz = khz.value
        self._out = torch.zeros(2, dtype=torch.int64, device="cuda")
        self._stream = torch.cuda.Stream()
        torch.cuda.synchronize()
        _lib.check(L.mcc_clock_probe(ctypes.c_void_p(self._stream.cuda_stream), ctypes.c_void_p(self._out.data_ptr()),
                                     16, float(seconds)))

    def mhz(self):
        self._stream.synchronize()
        wall, cycles = (int(v) for v in self._out.tolist())
        if wall <= 0:
            raise RuntimeError("clock probe has not run")
        return cycles / wall * self._khz / 1000.0

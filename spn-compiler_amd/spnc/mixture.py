"""Gated mixtures of compiled kernels on device-resident rows, ``p(x) = sum_j w_j(x) p_j(x)``: a sum node whose weights
depend on the row and of whose children every row visits a few.

``gate`` picks k experts a row and their weights, ``route`` sorts the rows' slots by expert, ``dispatch`` lays the rows out
in that order so that each expert reads one contiguous segment, and ``combine_log`` (log-likelihoods) or ``combine`` (rows of
activations) bring the experts' results back in row order with the weights applied. ``dropout`` marks features as missing
(NaN, for kernels compiled with ``supportMarginal``) or zeroes and scales activations. ``Mixture`` runs them around a list of
compiled kernels; ``HIPCompiler.compile_mixture`` builds one.

All take and return torch tensors on the GPU, run on the current stream, and have gradients where their inputs are
floating point (first order: a gradient cannot be differentiated again). Results do not change from run to run. Bad
arguments raise ``RuntimeError``. There is no CPU path.
"""
import math

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import spncpy

MAX_EXPERTS = 1024
MAX_CHOICES = 64

_TYPES = {torch.float32: 0, torch.float64: 1, torch.float16: 2, torch.bfloat16: 3}
_OVER = {"chosen": 0, "all": 1}
_LOG = 2
_ZERO, _MARGINAL, _MASK = 0, 1, 2
_LIMIT = 2 ** 31


def _refuse(condition, message):
    if condition:
        raise RuntimeError(message)


def _on_gpu(*tensors):
    """All tensors on one GPU; returns it."""
    device = tensors[0].device
    for t in tensors:
        _refuse(t.device.type != "cuda", f"Tensors must be on a GPU, got one on {t.device}")
        _refuse(t.device != device, f"Tensors must be on one GPU, got {device} and {t.device}")
    return device


def _call(name, device, *arguments):
    """Calls a function of the C-ABI on the device's current stream."""
    function = getattr(spncpy._load(), name)
    if torch.cuda.current_device() != device.index:
        with torch.cuda.device(device):
            spncpy._check(function(*arguments, torch.cuda.current_stream(device).cuda_stream))
    else:
        spncpy._check(function(*arguments, torch.cuda.current_stream(device).cuda_stream))


def _rows(t):
    """A 2-D tensor whose rows are contiguous and do not overlap; a copy where they are not."""
    n, width = t.shape
    if (width <= 1 or t.stride(1) == 1) and (n <= 1 or t.stride(0) >= width):
        return t
    return t.contiguous()


def _stride(t):
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _wants_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# ---- gate -----------------------------------------------------------------------------------------------------------

def _gate_forward(logits, k, flags):
    logits = _rows(logits)
    n, experts = logits.shape
    index = torch.empty((n, k), dtype=torch.int32, device=logits.device)
    weight = torch.empty((n, k), dtype=torch.float64 if logits.dtype == torch.float64 else torch.float32, device=logits.device)
    _call("spnc_hip_gate", logits.device, logits.data_ptr(), _TYPES[logits.dtype], n, experts, _stride(logits), k, flags, index.data_ptr(),
          weight.data_ptr())
    return index, weight


class _Gate(Function):
    @staticmethod
    def forward(ctx, logits, k, flags):
        index, weight = _gate_forward(logits, k, flags)
        ctx.flags, ctx.shape, ctx.dtype = flags, logits.shape, logits.dtype
        ctx.save_for_backward(logits if flags & 1 else None, index, weight)
        ctx.mark_non_differentiable(index)
        return index, weight

    @staticmethod
    @once_differentiable
    def backward(ctx, _, grad):
        logits, index, weight = ctx.saved_tensors
        (n, experts), k = ctx.shape, index.shape[1]
        logits = None if logits is None else _rows(logits)
        grad = grad.contiguous()
        out = torch.empty((n, experts), dtype=ctx.dtype, device=index.device)
        _call("spnc_hip_gate_backward", index.device, None if logits is None else logits.data_ptr(), _TYPES[ctx.dtype], n, experts,
              experts if logits is None else _stride(logits), k, ctx.flags, index.data_ptr(), weight.data_ptr(), grad.data_ptr(), out.data_ptr())
        return out, None, None


def gate(logits, k, *, over="chosen", log=False):
    """The k largest of a row's logits and their softmax weights.

    logits : [n, experts], float32, float64, float16 or bfloat16; at most 1024 experts.
    k      : choices a row, at most the number of experts and at most 64.
    over   : "chosen": the weights are a softmax over the chosen experts, "all": over all of them.
    log    : logarithms of the weights, for ``combine_log``.

    Returns ``(index, weight)``: int32 [n, k], by descending logit, equal ones by ascending index, NaN first; and the
    weights, float64 for float64 logits, else float32. Minus infinity closes an expert to a row: it is never chosen, and
    slots that are left over hold index -1 and weight 0 (log weight minus infinity). NaN among the logits makes the
    row's weights NaN if it is chosen, or anywhere in the row with "all".
    """
    _refuse(logits.dim() != 2, f"Logits must have shape [rows, experts], got {tuple(logits.shape)}")
    _refuse(logits.dtype not in _TYPES, f"Logits must be float32, float64, float16 or bfloat16, got {logits.dtype}")
    _refuse(over not in _OVER, f"over must be 'chosen' or 'all', got {over!r}")
    experts = logits.shape[1]
    _refuse(not 1 <= experts <= MAX_EXPERTS, f"The number of experts must be between 1 and {MAX_EXPERTS}, got {experts}")
    _refuse(not 1 <= k <= min(experts, MAX_CHOICES), f"k must be between 1 and {min(experts, MAX_CHOICES)}, got {k}")
    _on_gpu(logits)
    flags = _OVER[over] | (_LOG if log else 0)
    if _wants_grad(logits):
        return _Gate.apply(logits, k, flags)
    return _gate_forward(logits, k, flags)


# ---- routing --------------------------------------------------------------------------------------------------------

class Plan:
    """Where every slot (row i, choice j) stands in the buffer sorted by expert.

    position : int32 [n, k], the slot's row of the sorted buffer, -1 where it is not routed.
    starts   : int32 [experts + 1], first row of every expert's segment; the last entry is where the last segment ends.
    counts   : int32 [experts], rows of every segment.
    capacity : rows of the sorted buffer.
    """
    __slots__ = ("position", "starts", "counts", "capacity")

    def __init__(self, position, starts, counts, capacity):
        for name, t, dim in (("position", position, 2), ("starts", starts, 1), ("counts", counts, 1)):
            _refuse(t.dtype != torch.int32 or t.dim() != dim or not t.is_contiguous(), f"{name} must be a contiguous int32 tensor of {dim} dimensions")
        _refuse(position.shape[1] < 1, "A row must have at least one slot")
        _refuse(starts.shape[0] != counts.shape[0] + 1, "starts must have one entry more than counts")
        _refuse(not 1 <= counts.shape[0] <= MAX_EXPERTS, f"The number of experts must be between 1 and {MAX_EXPERTS}, got {counts.shape[0]}")
        _refuse(not 0 <= capacity < _LIMIT, f"The capacity must be below 2^31, got {capacity}")
        self.position, self.starts, self.counts, self.capacity = position, starts, counts, capacity

    @property
    def rows(self):
        return self.position.shape[0]

    @property
    def experts(self):
        return self.counts.shape[0]


def route(index, experts, *, align=1):
    """A stable sort of the slots by expert.

    index   : int32 [n, k], the expert of every slot, as ``gate`` returns it; anything outside [0, experts) is not routed. A
              row may name an expert twice.
    experts : their number, at most 1024.
    align   : segments start at multiples of this many rows (kernels want their input 16-byte aligned).

    Returns a ``Plan`` with capacity ``n * k + experts * (align - 1)``.
    """
    _refuse(index.dim() != 2 or index.dtype != torch.int32 or index.shape[1] < 1, f"The index must be int32 [rows, choices], got {index.dtype} {tuple(index.shape)}")
    _refuse(not 1 <= experts <= MAX_EXPERTS, f"The number of experts must be between 1 and {MAX_EXPERTS}, got {experts}")
    _refuse(align < 1, f"align must be at least 1, got {align}")
    slots = index.numel()
    capacity = slots + experts * (align - 1)
    _refuse(capacity >= _LIMIT, f"{slots} slots and {experts} segments aligned to {align} rows exceed 2^31 rows")
    device = _on_gpu(index)
    index = index.contiguous()
    position = torch.empty_like(index)
    starts = torch.empty(experts + 1, dtype=torch.int32, device=device)
    counts = torch.empty(experts, dtype=torch.int32, device=device)
    bytes_ = spncpy._load().spnc_hip_route_workspace(slots, experts)
    workspace = torch.empty(bytes_, dtype=torch.uint8, device=device) if bytes_ else None
    _call("spnc_hip_route", device, index.data_ptr(), slots, experts, align, position.data_ptr(), starts.data_ptr(), counts.data_ptr(),
          workspace.data_ptr() if bytes_ else None, bytes_)
    return Plan(position, starts, counts, capacity)


def _dispatch_forward(rows, plan, out, clear):
    rows = _rows(rows)
    n, width = rows.shape
    size = rows.element_size()
    if out is None:
        out = torch.empty((plan.capacity, width), dtype=rows.dtype, device=rows.device)
    _call("spnc_hip_dispatch", rows.device, rows.data_ptr(), n, width * size, _stride(rows) * size, plan.position.data_ptr(), plan.position.shape[1],
          plan.capacity, plan.starts.data_ptr(), plan.counts.data_ptr(), plan.experts, int(clear), out.data_ptr())
    return out


def _combine_forward(values, plan, weights):
    values = _rows(values)
    width = values.shape[1]
    out = torch.empty((plan.rows, width), dtype=values.dtype, device=values.device)
    _call("spnc_hip_combine", values.device, values.data_ptr(), _TYPES[values.dtype], plan.capacity, width, _stride(values), plan.position.data_ptr(),
          plan.rows, plan.position.shape[1], None if weights is None else weights.data_ptr(), 0 if weights is None else _TYPES[weights.dtype],
          out.data_ptr())
    return out


class _Dispatch(Function):
    @staticmethod
    def forward(ctx, rows, plan):
        ctx.plan = plan
        ctx.save_for_backward(plan.position)
        return _dispatch_forward(rows, plan, None, True)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        ctx.saved_tensors  # raises if the plan was written to in the meantime
        return _combine_forward(grad, ctx.plan, None), None


def dispatch(rows, plan, out=None):
    """The rows in the plan's order: ``out[plan.position[i, j]] = rows[i]`` for every slot that is routed.

    rows : [n, width] of any type of 1, 2, 4 or 8 bytes an element; differentiable where floating point.
    out  : [capacity, width] to write into; its rows that belong to no segment are left as they were. Without it a new
           tensor is returned in which they are zero.
    """
    _refuse(rows.dim() != 2, f"Rows must have shape [rows, width], got {tuple(rows.shape)}")
    _refuse(rows.shape[0] != plan.rows, f"The plan is for {plan.rows} rows, got {rows.shape[0]}")
    _refuse(rows.element_size() not in (1, 2, 4, 8) or rows.dtype.is_complex, f"Rows of {rows.dtype} are not supported")
    if out is not None:
        _refuse(tuple(out.shape) != (plan.capacity, rows.shape[1]) or out.dtype != rows.dtype or not out.is_contiguous(),
                f"out must be a contiguous {rows.dtype} tensor of shape {(plan.capacity, rows.shape[1])}")
        _refuse(_wants_grad(rows, out), "dispatch with out= has no gradient; call it without")
        _on_gpu(rows, plan.position, plan.starts, plan.counts, out)
        return _dispatch_forward(rows, plan, out, False)
    _on_gpu(rows, plan.position, plan.starts, plan.counts)
    if _wants_grad(rows):
        _refuse(rows.dtype not in _TYPES, f"Rows of {rows.dtype} have no gradient")
        return _Dispatch.apply(rows, plan)
    return _dispatch_forward(rows, plan, None, True)


# ---- combination ----------------------------------------------------------------------------------------------------

class _Combine(Function):
    @staticmethod
    def forward(ctx, values, weights, plan):
        ctx.plan = plan
        ctx.save_for_backward(values, weights, plan.position)
        return _combine_forward(values, plan, weights)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        values, weights, position = ctx.saved_tensors
        plan, values, grad = ctx.plan, _rows(values), _rows(grad)
        width = values.shape[1]
        if weights is None:
            return _dispatch_forward(grad, plan, None, True), None, None
        grad_values = torch.empty((plan.capacity, width), dtype=values.dtype, device=values.device) if ctx.needs_input_grad[0] else None
        grad_weights = torch.empty_like(weights) if ctx.needs_input_grad[1] else None
        _call("spnc_hip_combine_backward", values.device, values.data_ptr(), _TYPES[values.dtype], plan.capacity, width, _stride(values),
              position.data_ptr(), plan.rows, position.shape[1], weights.data_ptr(), _TYPES[weights.dtype], grad.data_ptr(), _stride(grad),
              plan.starts.data_ptr(), plan.counts.data_ptr(), plan.experts, None if grad_values is None else grad_values.data_ptr(),
              None if grad_weights is None else grad_weights.data_ptr())
        return grad_values, grad_weights, None


def _check_weights(weights, plan, allowed):
    _refuse(tuple(weights.shape) != tuple(plan.position.shape), f"Weights must have shape {tuple(plan.position.shape)}, got {tuple(weights.shape)}")
    _refuse(weights.dtype not in allowed, f"Weights must be {' or '.join(str(t) for t in allowed)}, got {weights.dtype}")


def combine(values, plan, weights=None):
    """Rows of the sorted buffer back in row order, weighted: ``out[i] = sum_j weights[i, j] * values[plan.position[i, j]]``.

    values  : [capacity, width], float32, float64, float16 or bfloat16; sums are held in 32 bits (64 for float64).
    weights : [n, k], float32, or float64 with float64 values; None for ones. Differentiable, as the values are.

    Slots that are not routed are left out; a row without slots becomes zero.
    """
    _refuse(values.dim() != 2 or values.shape[0] != plan.capacity, f"Values must have shape [{plan.capacity}, width], got {tuple(values.shape)}")
    _refuse(values.dtype not in _TYPES, f"Values must be float32, float64, float16 or bfloat16, got {values.dtype}")
    if weights is None:
        _on_gpu(values, plan.position, plan.starts, plan.counts)
    else:
        _check_weights(weights, plan, (torch.float32, torch.float64) if values.dtype == torch.float64 else (torch.float32,))
        _on_gpu(values, plan.position, plan.starts, plan.counts, weights)
        weights = weights.contiguous()
    if _wants_grad(values, weights):
        return _Combine.apply(values, weights, plan)
    return _combine_forward(values, plan, weights)


def _combine_log_forward(values, plan, weights):
    out = torch.empty(plan.rows, dtype=values.dtype, device=values.device)
    _call("spnc_hip_combine_log", values.device, values.data_ptr(), _TYPES[values.dtype], plan.capacity, plan.position.data_ptr(), plan.rows,
          plan.position.shape[1], weights.data_ptr(), _TYPES[weights.dtype], out.data_ptr())
    return out


class _CombineLog(Function):
    @staticmethod
    def forward(ctx, values, weights, plan):
        ctx.plan = plan
        ctx.save_for_backward(values, weights, plan.position)
        return _combine_log_forward(values, plan, weights)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        values, weights, position = ctx.saved_tensors
        plan, grad = ctx.plan, grad.contiguous()
        grad_values = torch.empty_like(values) if ctx.needs_input_grad[0] else None
        grad_weights = torch.empty_like(weights) if ctx.needs_input_grad[1] else None
        _call("spnc_hip_combine_log_backward", values.device, values.data_ptr(), _TYPES[values.dtype], plan.capacity, position.data_ptr(), plan.rows,
              position.shape[1], weights.data_ptr(), _TYPES[weights.dtype], grad.data_ptr(), plan.starts.data_ptr(), plan.counts.data_ptr(),
              plan.experts, None if grad_values is None else grad_values.data_ptr(), None if grad_weights is None else grad_weights.data_ptr())
        return grad_values, grad_weights, None


def combine_log(values, plan, log_weights):
    """Log-likelihoods of the sorted rows joined into the mixture's: ``out[i] = log sum_j exp(log_weights[i, j] +
    values[plan.position[i, j]])``.

    values      : [capacity], float32 or float64, one a row of the sorted buffer.
    log_weights : [n, k], float32 or float64. Both are differentiable.

    A slot that is not routed, or whose log weight is minus infinity, is left out whatever its value is; a row without
    slots, or all of whose values are minus infinity, becomes minus infinity and has no gradient.
    """
    _refuse(values.dim() != 1 or values.shape[0] != plan.capacity, f"Values must have shape [{plan.capacity}], got {tuple(values.shape)}")
    _refuse(values.dtype not in (torch.float32, torch.float64), f"Values must be float32 or float64, got {values.dtype}")
    _check_weights(log_weights, plan, (torch.float32, torch.float64))
    _on_gpu(values, plan.position, plan.starts, plan.counts, log_weights)
    values, log_weights = values.contiguous(), log_weights.contiguous()
    if _wants_grad(values, log_weights):
        return _CombineLog.apply(values, log_weights, plan)
    return _combine_log_forward(values, plan, log_weights)


# ---- dropout --------------------------------------------------------------------------------------------------------

def _dropout_forward(x, p, mode, seed, offset):
    shape = x.shape
    if x.dim() != 2:
        x = x.reshape(1, -1) if x.dim() < 2 else x.reshape(-1, shape[-1])
    x = _rows(x)
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    on_device = isinstance(offset, torch.Tensor)
    _call("spnc_hip_dropout", x.device, x.data_ptr(), _TYPES[x.dtype], x.shape[0], x.shape[1], _stride(x), out.data_ptr(), x.shape[1], p, mode, seed,
          0 if on_device else offset, offset.data_ptr() if on_device else None)
    return out.view(shape)


class _Dropout(Function):
    @staticmethod
    def forward(ctx, x, p, mode, seed, offset):
        ctx.arguments = p, mode, seed
        on_device = isinstance(offset, torch.Tensor)
        ctx.save_for_backward(offset if on_device else None)  # the mask must be the same: a change in between is an error
        ctx.offset = None if on_device else offset
        return _dropout_forward(x, p, mode, seed, offset)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        (offset,), (p, mode, seed) = ctx.saved_tensors, ctx.arguments
        return _dropout_forward(grad, p, _MASK if mode == _MARGINAL else mode, seed, ctx.offset if offset is None else offset), None, None, None, None


def dropout(x, p, seed, *, offset=0, marginal=False):
    """Drops every element of x with probability p; the mask comes from a counter-based generator and is never stored.

    x        : any shape, float32, float64, float16 or bfloat16.
    seed     : 0 <= seed < 2^64.
    offset   : tells calls of one seed apart; 0 <= offset < 2^64, or a one-element int64 tensor on the GPU, which a captured
               graph reads at every replay (do not write to it between a forward and its backward pass).
    marginal : False: dropped elements become 0, the others are multiplied by 1 / (1 - p). True: dropped elements become NaN, a
               missing feature to a kernel compiled with ``supportMarginal``, the others stay as they are.

    Element e of x, counted in its logical order whatever the strides and the type are, is dropped where word e % 4 of
    Philox4x32-10 with the seed as key and (e // 4, offset) as counter is below round(p * 2^32).
    """
    _refuse(x.dtype not in _TYPES, f"x must be float32, float64, float16 or bfloat16, got {x.dtype}")
    _refuse(not 0.0 <= p <= 1.0, f"p must be between 0 and 1, got {p}")
    _refuse(not 0 <= seed < 2 ** 64, f"The seed must be between 0 and 2^64 - 1, got {seed}")
    if isinstance(offset, torch.Tensor):
        _refuse(offset.dtype != torch.int64 or offset.numel() != 1, "An offset on the device must be a one-element int64 tensor")
        _on_gpu(x, offset)
    else:
        _refuse(not 0 <= offset < 2 ** 64, f"The offset must be between 0 and 2^64 - 1, got {offset}")
        _on_gpu(x)
    mode = _MARGINAL if marginal else _ZERO
    if _wants_grad(x):
        return _Dropout.apply(x, p, mode, seed, offset)
    return _dropout_forward(x, p, mode, seed, offset)


# ---- mixtures of kernels --------------------------------------------------------------------------------------------

class Mixture:
    """A gated mixture whose experts are compiled kernels (``HIPCompiler.compile_ll``) over the same features."""

    def __init__(self, kernels):
        self.kernels = list(kernels)
        _refuse(not 1 <= len(self.kernels) <= MAX_EXPERTS, f"The number of kernels must be between 1 and {MAX_EXPERTS}, got {len(self.kernels)}")
        infos = [k.info() for k in self.kernels]
        for key, what in (("num_features", "number of features"), ("bytes_per_feature", "feature type"), ("feature_is_float", "feature type"),
                          ("dtype", "result type")):
            values = sorted({i[key] for i in infos})
            _refuse(len(values) != 1, f"The kernels of a mixture must agree on the {what}, got {values}")
        self.num_features = infos[0]["num_features"]
        self._feature_bytes, self._feature_is_float = infos[0]["bytes_per_feature"], bool(infos[0]["feature_is_float"])
        self._result = torch.float32 if infos[0]["dtype"] == "float32" else torch.float64
        row_bytes = self.num_features * self._feature_bytes
        self._align = 1
        for i in infos:
            self._align = math.lcm(self._align, i["input_alignment"] // math.gcd(i["input_alignment"], row_bytes))

    def execute(self, rows, plan):
        """Log-likelihoods [plan.capacity] of sorted rows, each segment under its kernel; rows of no segment stay undefined.
        Waits for the plan: the host needs the segments' sizes to launch the kernels."""
        _refuse(tuple(rows.shape) != (plan.capacity, self.num_features) or not rows.is_contiguous(),
                f"Sorted rows must be contiguous with shape {(plan.capacity, self.num_features)}, got {tuple(rows.shape)}")
        _refuse(plan.experts != len(self.kernels), f"The plan is for {plan.experts} experts, the mixture has {len(self.kernels)}")
        self._check_type(rows)
        device = _on_gpu(rows, plan.position, plan.starts, plan.counts)
        _refuse(torch.cuda.is_current_stream_capturing(), "A mixture cannot run under graph capture: the host needs the segments' sizes")
        values = torch.empty(plan.capacity, dtype=self._result, device=device)
        row_bytes, result_bytes = self.num_features * self._feature_bytes, values.element_size()
        with torch.cuda.device(device):
            sizes = torch.cat((plan.starts, plan.counts)).tolist()
            stream = torch.cuda.current_stream(device).cuda_stream
            for e, kernel in enumerate(self.kernels):
                start, count = sizes[e], sizes[plan.experts + 1 + e]
                _refuse(start < 0 or count < 0 or start + count > plan.capacity, f"Segment {e} of the plan lies outside the sorted buffer")
                if count:
                    kernel.execute_device(count, rows.data_ptr() + start * row_bytes, values.data_ptr() + start * result_bytes, stream)
        return values

    def _check_type(self, rows):
        kind = rows.dtype.is_floating_point
        _refuse(rows.element_size() != self._feature_bytes or kind != self._feature_is_float or rows.dtype in (torch.bool, torch.bfloat16, torch.float16)
                or rows.dtype.is_complex,
                f"Rows of {rows.dtype} do not match the kernels' feature type {'float' if self._feature_is_float else 'int'}{8 * self._feature_bytes}")

    def log_likelihood(self, rows, logits, k, *, over="chosen"):
        """Log-likelihood [n] of every row under the mixture of its k best experts, differentiable in the logits.

        rows   : [n, features] of the kernels' feature type.
        logits : [n, kernels] of the gate, see ``gate`` for ``k`` and ``over``.
        """
        _refuse(rows.dim() != 2 or rows.shape[1] != self.num_features, f"Rows must have shape [rows, {self.num_features}], got {tuple(rows.shape)}")
        _refuse(logits.dim() != 2 or tuple(logits.shape) != (rows.shape[0], len(self.kernels)),
                f"Logits must have shape [{rows.shape[0]}, {len(self.kernels)}], got {tuple(logits.shape)}")
        self._check_type(rows)
        _refuse(_wants_grad(rows), "Compiled kernels have no gradient with respect to their features")
        device = _on_gpu(rows, logits)
        index, log_weights = gate(logits, k, over=over, log=True)
        plan = route(index, len(self.kernels), align=self._align)
        sorted_rows = torch.empty((plan.capacity, self.num_features), dtype=rows.dtype, device=device)
        return combine_log(self.execute(dispatch(rows, plan, out=sorted_rows), plan), plan, log_weights)

"""Gated mixtures of compiled kernels on device-resident rows, ``p(x) = sum_j w_j(x) p_j(x)``: a sum node whose weights
depend on the row and of whose children every row visits a few.

``gate`` picks k experts a row and their weights, ``route`` sorts the rows' slots by expert, ``dispatch`` lays the rows out
in that order so that each expert reads one contiguous segment, and ``combine_log`` (log-likelihoods) or ``combine`` (rows of
activations) bring the experts' results back in row order with the weights applied. ``dropout`` marks features as missing
(NaN, for kernels compiled with ``supportMarginal``) or zeroes and scales activations. ``Mixture`` runs them around a list of
compiled kernels; ``HIPCompiler.compile_mixture`` builds one.

All take and return torch tensors on the GPU, run on the current stream, and have gradients where their inputs are
floating point (first order: a gradient cannot be differentiated again; there are no forward-mode derivatives). Results do
not change from run to run. Bad arguments raise ``RuntimeError``, and so do calls under ``torch.jit.trace``, ``make_fx`` or
``torch.export``, which would record nothing of them. An error that an earlier HIP call of the thread left unread is told as a
warning. There is no CPU path.
"""
import math

import torch

from . import spncpy

MAX_EXPERTS = 1024
MAX_CHOICES = 64

_OVER = {"chosen": 0, "all": 1}
_LOG = 2
_native = None


def _ops():
    """The native half (csrc/torch_binding.cpp). It finds libspnc_hip.so already loaded, by the way every user of it takes."""
    global _native
    if _native is None:
        spncpy._load()
        try:
            from . import _mixture_ops
        except ImportError as e:
            raise RuntimeError(f"The native part of spnc.mixture is missing; build it with `make -C spn-compiler_amd/csrc` ({e})") from e
        _native = _mixture_ops
    return _native


def _refuse(condition, message):
    if condition:
        raise RuntimeError(message)


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
    _refuse(over not in _OVER, f"over must be 'chosen' or 'all', got {over!r}")
    return (_native or _ops()).gate(logits, k, _OVER[over] | (_LOG if log else 0))


class Plan:
    """Where every slot (row i, choice j) stands in the buffer sorted by expert.

    position : int32 [n, k], the slot's row of the sorted buffer, -1 where it is not routed; a row of the buffer belongs to one slot.
    starts   : int32 [experts + 1], first row of every expert's segment; the last entry is where the last segment ends.
    counts   : int32 [experts], rows of every segment.
    capacity : rows of the sorted buffer.
    """
    __slots__ = ("position", "starts", "counts", "capacity")

    def __init__(self, position, starts, counts, capacity):
        (_native or _ops()).check_plan(position, starts, counts, capacity)
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
    plan = Plan.__new__(Plan)
    plan.position, plan.starts, plan.counts, plan.capacity = (_native or _ops()).route(index, experts, align)
    return plan


def dispatch(rows, plan, out=None):
    """The rows in the plan's order: ``out[plan.position[i, j]] = rows[i]`` for every slot that is routed.

    rows : [n, width] of any type of 1, 2, 4 or 8 bytes an element; differentiable where floating point.
    out  : [capacity, width] to write into, which must not share memory with rows or plan; its rows that belong to no segment are left
           as they were. Without it a new tensor is returned in which they are zero.
    """
    return (_native or _ops()).dispatch(rows, plan.position, plan.starts, plan.counts, plan.capacity, out)


def combine(values, plan, weights=None):
    """Rows of the sorted buffer back in row order, weighted: ``out[i] = sum_j weights[i, j] * values[plan.position[i, j]]``.

    values  : [capacity, width], float32, float64, float16 or bfloat16; sums are held in 32 bits (64 for float64).
    weights : [n, k], float32, or float64 with float64 values; None for ones. Differentiable, as the values are.

    Slots that are not routed are left out; a row without slots becomes zero.
    """
    return (_native or _ops()).combine(values, plan.position, plan.starts, plan.counts, plan.capacity, weights)


def combine_log(values, plan, log_weights):
    """Log-likelihoods of the sorted rows joined into the mixture's: ``out[i] = log sum_j exp(log_weights[i, j] +
    values[plan.position[i, j]])``.

    values      : [capacity], float32 or float64, one a row of the sorted buffer.
    log_weights : [n, k], float32 or float64. Both are differentiable.

    A slot that is not routed, or whose log weight is minus infinity, is left out whatever its value is; a row without
    slots, or all of whose values are minus infinity, becomes minus infinity and has no gradient.
    """
    return (_native or _ops()).combine_log(values, plan.position, plan.starts, plan.counts, plan.capacity, log_weights)


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
    _refuse(not 0.0 <= p <= 1.0, f"p must be between 0 and 1, got {p}")
    _refuse(not 0 <= seed < 2 ** 64, f"The seed must be between 0 and 2^64 - 1, got {seed}")
    if isinstance(offset, torch.Tensor):
        return (_native or _ops()).dropout(x, p, seed, 0, offset, marginal)
    _refuse(not 0 <= offset < 2 ** 64, f"The offset must be between 0 and 2^64 - 1, got {offset}")
    return (_native or _ops()).dropout(x, p, seed, offset, None, marginal)


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
        self._side = {}

    def _lanes(self, device):
        """The current stream and three others, made once a device. Segments are short and their kernels long chains that leave most of
        the chip free: a call of ten 16-feature kernels over 4096 rows takes 211 us this way and 223 one after the other, over 1 M rows
        384 and 428, the wait for the segments' sizes included; over 30 rows 220 and 191, since there the host's launches are all of it."""
        if device not in self._side:
            self._side[device] = [torch.cuda.Stream(device) for _ in range(3)]
        return [torch.cuda.current_stream(device)] + self._side[device]

    def execute(self, rows, plan):
        """Log-likelihoods [plan.capacity] of sorted rows, each segment under its kernel; rows of no segment stay undefined.
        Kernels have no gradient with respect to their features: rows that want one are refused. Waits for the plan: the host needs the segments' sizes to launch the kernels."""
        self._check_derivatives(rows)
        _refuse(tuple(rows.shape) != (plan.capacity, self.num_features) or not rows.is_contiguous(),
                f"Sorted rows must be contiguous with shape {(plan.capacity, self.num_features)}, got {tuple(rows.shape)}")
        _refuse(plan.experts != len(self.kernels), f"The plan is for {plan.experts} experts, the mixture has {len(self.kernels)}")
        self._check_type(rows)
        device = rows.device
        _refuse(device.type != "cuda" or any(t.device != device for t in (plan.position, plan.starts, plan.counts)),
                f"Rows and plan must be on one GPU, got {device} and {plan.position.device}")
        _refuse(torch.cuda.is_current_stream_capturing(), "A mixture cannot run under graph capture: the host needs the segments' sizes")
        rows = rows.resolve_neg()
        values = torch.empty(plan.capacity, dtype=self._result, device=device)
        row_bytes, result_bytes = self.num_features * self._feature_bytes, values.element_size()
        with torch.cuda.device(device):
            sizes = torch.cat((plan.starts, plan.counts)).tolist()
            segments = []
            for e in range(plan.experts):
                start, count = sizes[e], sizes[plan.experts + 1 + e]
                _refuse(start < 0 or count < 0 or start + count > plan.capacity, f"Segment {e} of the plan lies outside the sorted buffer")
                if count:
                    segments.append((count, start, self.kernels[e]))
            segments.sort(key=lambda segment: -segment[0])      # the long ones first, each on the next stream
            lanes = self._lanes(device) if len(segments) >= 4 else [torch.cuda.current_stream(device)]
            for lane in lanes[1:]:
                lane.wait_stream(lanes[0])
            try:
                for i, (count, start, kernel) in enumerate(segments):
                    kernel.execute_device(count, rows.data_ptr() + start * row_bytes, values.data_ptr() + start * result_bytes,
                                          lanes[i % len(lanes)].cuda_stream)
            finally:
                for lane in lanes[1:]:
                    lanes[0].wait_stream(lane)
        return values

    @staticmethod
    def _check_derivatives(rows):
        _refuse(torch.is_grad_enabled() and rows.requires_grad, "Compiled kernels have no gradient with respect to their features")
        _ops().check_recorded(rows)

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
        self._check_derivatives(rows)
        _ops().check_recorded(logits)
        _refuse(rows.dim() != 2 or rows.shape[1] != self.num_features, f"Rows must have shape [rows, {self.num_features}], got {tuple(rows.shape)}")
        _refuse(logits.dim() != 2 or tuple(logits.shape) != (rows.shape[0], len(self.kernels)),
                f"Logits must have shape [{rows.shape[0]}, {len(self.kernels)}], got {tuple(logits.shape)}")
        self._check_type(rows)
        _refuse(rows.device.type != "cuda" or logits.device != rows.device, f"Rows and logits must be on one GPU, got {rows.device} and {logits.device}")
        index, log_weights = gate(logits, k, over=over, log=True)
        plan = route(index, len(self.kernels), align=self._align)
        sorted_rows = torch.empty((plan.capacity, self.num_features), dtype=rows.dtype, device=rows.device)
        return combine_log(self.execute(dispatch(rows, plan, out=sorted_rows), plan), plan, log_weights)

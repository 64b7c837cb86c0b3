"""Orthogonalised updates on gfx950: Newton-Schulz products, and Muon with a stored-format momentum.

``orthogonalize`` brings the singular values of a matrix near one by
Newton-Schulz products; ``MuonHip`` and ``hip_muon_step_`` update 2-D weights by
the orthogonalised momentum, which is stored in any of this package's formats
with its random streams (``momentum_buffer``, as ``SGDMHip`` stores it).  The
reference package has no counterpart.
"""

from __future__ import annotations

import math
from functools import lru_cache

import numpy as np
import torch

from .. import _lib
from .._hash import update_key
from ..optim._dtensor import is_dtensor
from ..optim._state import StateOptimizer
from ..rounding import native_codes
from ._common import validate_device
from ._optimizer import (
    DEFAULT_BLOCK_SIZE,
    nonnegative,
    reject_dtensors,
    resolve_native_codes,
    validate_no_overlap,
    validate_tensor_layout,
)

_STATE_NAMES = ("momentum_buffer",)
_DTYPES = (torch.float32, torch.bfloat16, torch.float16)
# The quintic whose slope at zero is largest while every singular value in
# [0, 1] ends near 1 after five steps.
NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)
NS_STEPS = 5
NS_EPS = 1e-7
UPDATE_SCALES = ("spectral", "rms")
# Bounds of the scaled FP16 operands (sr_matrix_hip.h, sr_newton_schulz).
_MAX_SINGULAR, _MAX_POLYNOMIAL, _SHIFT = 2.5, 7.0, 1.5
# A launch's workspace: larger batches are updated in turn.
_WORKSPACE_BYTES = 4 << 30


@lru_cache(maxsize=64)
def _newton_schulz(steps: int, coefficients: tuple, eps: float) -> _lib.NewtonSchulz:
    """The checked C record of an iteration.

    The products' FP16 operands leave room for singular values up to 2.5 and
    for b s^2 + c s^4 up to 5.5, so the iterates of every singular value of
    a normalized matrix, in [0, 1], must stay inside.
    """
    if isinstance(steps, bool) or not isinstance(steps, int) or steps < 1:
        raise ValueError(f"steps must be a positive integer, not {steps!r}")
    if len(coefficients) != 3 or not all(math.isfinite(c) for c in coefficients):
        raise ValueError("coefficients must be three finite numbers")
    if not math.isfinite(eps) or eps < 0:
        raise ValueError(f"invalid eps: {eps}")
    a, b, c = coefficients
    s = np.linspace(0.0, 1.0, 4097)
    for _ in range(steps):
        polynomial = b * s**2 + c * s**4
        if s.max() > _MAX_SINGULAR or np.abs(polynomial).max() + _SHIFT > _MAX_POLYNOMIAL:
            raise ValueError(f"coefficients {coefficients} take singular values out of range in {steps} steps")
        s = np.abs(s * (a + polynomial))
    return _lib.NewtonSchulz(a, b, c, eps, steps)


def _batch_size(count: int, rows: int, cols: int) -> int:
    """Matrices of ``count`` per launch: as many as the library takes, within the workspace's limit."""
    one = _lib.library().sr_orthogonalize_workspace(1, rows, cols)
    return max(1, min(count, _lib.MATRIX_BATCH, _WORKSPACE_BYTES // max(one, 1)))


def _workspace_bytes(count: int, rows: int, cols: int) -> int:
    """Bytes of workspace of the launches that update ``count`` matrices; raises for matrices the library refuses."""
    size = _lib.library().sr_orthogonalize_workspace(_batch_size(count, rows, cols), rows, cols)
    if not size:
        raise ValueError(f"{rows} x {cols} matrices are too large")
    return size


def orthogonalize(
    x: torch.Tensor,
    *,
    steps: int = NS_STEPS,
    coefficients: tuple = NS_COEFFICIENTS,
    eps: float = NS_EPS,
    dtype: torch.dtype = torch.bfloat16,
) -> torch.Tensor:
    """The orthogonalised matrices of ``x`` (..., rows, cols), by Newton-Schulz products.

    Each matrix X is divided by its Frobenius norm plus ``eps``; then ``steps``
    times X <- a X + (b G + c G^2) X with G = X X^T (on the smaller side).  The
    default coefficients bring the singular values of most matrices into about
    [0.7, 1.2]; a matrix of zeros stays zero.

    ``x`` is FP32, BF16 or FP16 on the GPU; ``dtype`` is the result's.  The
    products take FP16 operands and sum in FP32: the result is within about
    2e-3 (relative, Frobenius norm) of the exact iteration, which BF16 holds.
    Matrices that are not contiguous are copied first.  Nothing is recorded
    for autograd.
    """
    reject_dtensors(x)
    if dtype not in _DTYPES:
        raise TypeError(f"dtype must be FP32, BF16 or FP16, not {dtype}")
    ns = _newton_schulz(steps, tuple(coefficients), float(eps))
    device = getattr(x, "device", None)
    stream = 0
    if device is not None and device.type == "cuda":  # the native entry refuses everything else
        validate_device(device)
        stream = _lib.stream_handle(device)
    out = _lib.matrix().orthogonalize(
        x, _lib.DTYPE_CODES[dtype], ns.a, ns.b, ns.c, ns.eps, ns.steps, _WORKSPACE_BYTES, stream
    )
    if not isinstance(out, torch.Tensor):
        _lib.check("sr_orthogonalize", out)
    return out


def _update_scale(kind: str, rows: int, cols: int) -> float:
    """The factor on the learning rate for a rows x cols update."""
    return math.sqrt(max(1.0, rows / cols)) if kind == "spectral" else 0.2 * math.sqrt(max(rows, cols))


def _matrix_shape(parameter) -> tuple:
    """The matrix a parameter is orthogonalised as: its first dimension by the others together."""
    if parameter.dim() < 2:
        raise ValueError("Muon updates matrices: pass parameters of one dimension to another optimizer")
    rows = parameter.shape[0]
    return rows, parameter.numel() // rows if rows else 0


def _validate_hyper(lr, momentum, weight_decay, update_scale):
    nonnegative("learning rate", lr)
    if not 0 <= momentum < 1:
        raise ValueError(f"invalid momentum value: {momentum}")
    nonnegative("weight_decay", weight_decay)
    if update_scale not in UPDATE_SCALES:
        raise ValueError(f"update_scale must be one of {UPDATE_SCALES}")


def _launch(tensors, shape, keys, codes, hyper, ns, workspace):
    """Queue the update of same-shaped (parameter, gradient, momentum) rows; keys are (key, offset)."""
    lr, momentum, nesterov, weight_decay, update_scale = hyper
    parameter, gradient, _ = tensors[0]
    code, rule = codes
    rows, cols = shape
    hparams = _lib.MuonHparams(
        momentum, 1 - lr * weight_decay, -lr * _update_scale(update_scale, rows, cols), int(nesterov)
    )
    device = workspace.device
    each = _batch_size(len(tensors), rows, cols)
    with _lib.on_device(device):
        for first in range(0, len(tensors), each):
            part = range(first, min(first + each, len(tensors)))
            table = (_lib.MuonRow * len(part))(
                *((*(t.data_ptr() for t in tensors[i]), *keys[i]) for i in part)
            )
            _lib.call(
                "sr_muon_multi", table, len(part), rows, cols, _lib.DTYPE_CODES[parameter.dtype],
                _lib.DTYPE_CODES[gradient.dtype], code, rule, hparams, ns, workspace.data_ptr(),
                _lib.stream_handle(device),
            )


def _spans(tensors):
    for role, t in enumerate(tensors):
        start = t.data_ptr()
        yield start, start + t.numel() * t.element_size(), role != 1


def hip_muon_step_(
    parameter: torch.Tensor,
    gradient: torch.Tensor,
    momentum: torch.Tensor,
    *,
    lr: float,
    momentum_factor: float,
    nesterov: bool = True,
    weight_decay: float = 0.0,
    update_scale: str = "spectral",
    ns_steps: int = NS_STEPS,
    ns_coefficients: tuple = NS_COEFFICIENTS,
    eps: float = NS_EPS,
    seed: int,
    offset: int = 0,
    rounding: str | None = None,
    formats: tuple | dict | None = None,
) -> None:
    """Apply one Muon update to a matrix in place.

    With u the momentum and f = ``momentum_factor``:

    - ``u = f * u + gradient``, stored in the momentum's format with the
      random stream ``state_key(seed, 0)`` from ``offset`` on;
    - ``o = orthogonalize(gradient + f * u)`` with ``nesterov``, else of u
      (u before its rounding);
    - ``parameter = parameter * (1 - lr * weight_decay) - lr * s * o``, where s
      is sqrt(max(1, rows / cols)) ("spectral") or 0.2 sqrt(max(rows, cols))
      ("rms", which matches the size of AdamW's updates).

    The three tensors are same-shaped, contiguous and on one GPU; parameter and
    gradient FP32 or BF16, the momentum in any built-in storage format.  More
    than two dimensions are taken as the first by all others.
    """
    grad = torch.is_grad_enabled()
    _lib.set_grad_enabled(False)
    try:
        codes = resolve_native_codes(_STATE_NAMES, (momentum,), formats, rounding, DEFAULT_BLOCK_SIZE)
        _validate_hyper(lr, momentum_factor, weight_decay, update_scale)
        ns = _newton_schulz(ns_steps, tuple(ns_coefficients), float(eps))
        tensors = (parameter, gradient, momentum)
        reject_dtensors(*tensors)
        validate_tensor_layout(tensors)
        shape = _matrix_shape(parameter)
        device = parameter.device
        validate_device(device)
        validate_no_overlap(_spans(tensors))
        if parameter.numel():
            workspace = torch.empty(_workspace_bytes(1, *shape), dtype=torch.uint8, device=device)
            _launch([tensors], shape, [(_lib.low32(seed), _lib.low32(offset))], codes[0],
                    (lr, momentum_factor, nesterov, weight_decay, update_scale), ns, workspace)
    finally:
        _lib.set_grad_enabled(grad)


class MuonHip(StateOptimizer):
    """Muon: orthogonalised momentum updates of matrices, BF16 stochastic momentum storage by default.

    For parameters of at least two dimensions (others, and usually embeddings
    and heads, belong to :class:`AdamWHip`); more than two are taken as the
    first by all others.  Parameters of one shape and dtype are updated
    together.  See :func:`hip_muon_step_` for the update and the arguments; the
    state is ``momentum_buffer`` and each update's key is
    ``update_key(seed, rng_step, parameter index)``, as in ``SGDMHip``.
    DTensor parameters are refused: the update needs whole matrices.
    """

    _state_names = _STATE_NAMES
    _uses_step = False
    _rounding_backend = "hip"

    def __init__(
        self,
        params,
        lr=0.02,
        momentum=0.95,
        *,
        nesterov=True,
        weight_decay=0.0,
        update_scale="spectral",
        ns_steps=NS_STEPS,
        ns_coefficients=NS_COEFFICIENTS,
        eps=NS_EPS,
        state_format=None,
        state_dtype=None,
        rounding=None,
        seed=0,
    ):
        super().__init__(
            params,
            {
                "lr": lr,
                "momentum": momentum,
                "nesterov": nesterov,
                "weight_decay": weight_decay,
                "update_scale": update_scale,
                "ns_steps": ns_steps,
                "ns_coefficients": tuple(ns_coefficients),
                "eps": eps,
            },
            state_format=state_format,
            state_dtype=state_dtype,
            rounding=rounding,
            seed=seed,
        )

    def _validate_group(self, group):
        _validate_hyper(group["lr"], group["momentum"], group["weight_decay"], group["update_scale"])
        _newton_schulz(group["ns_steps"], tuple(group["ns_coefficients"]), float(group["eps"]))

    def add_param_group(self, param_group):
        params = param_group["params"]
        if isinstance(params, torch.Tensor):
            params = [params]
        elif not isinstance(params, set):  # which torch refuses, below
            params = list(params)
        for parameter in params:
            # Named parameters come as (name, parameter).
            matrix = parameter[1] if isinstance(parameter, tuple) else parameter
            if isinstance(matrix, torch.Tensor):
                _matrix_shape(matrix)
        super().add_param_group({**param_group, "params": params})

    def _shard_start(self, parameter):
        if is_dtensor(parameter):
            raise NotImplementedError("MuonHip needs whole matrices, not DTensor shards")
        return 0

    def _hyper(self, group):
        return group["lr"], group["momentum"], group["nesterov"], group["weight_decay"], group["update_scale"]

    def _step_group(self, group, formats, items, rng_step):
        if _lib.capturing():
            raise RuntimeError(
                f"{type(self).__name__}.step() cannot be captured in a HIP graph: each step's learning rate and RNG "
                "step are kernel arguments, which a graph replay would repeat"
            )
        _validate_hyper(*(group[name] for name in ("lr", "momentum", "weight_decay", "update_scale")))
        ns = _newton_schulz(group["ns_steps"], tuple(group["ns_coefficients"]), float(group["eps"]))
        codes = native_codes(formats[0].dtype, formats[0].rounding)
        # The whole group is checked, and its workspaces are there, before its first launch: a step that is refused or
        # runs out of memory has changed nothing.
        buckets, spans = {}, {}
        for parameter, state, index, _, offset in items:
            tensors = (parameter, parameter.grad, state["momentum_buffer"])
            validate_tensor_layout(tensors)
            if not parameter.numel():
                continue
            device = parameter.device
            validate_device(device)
            spans.setdefault(device, []).extend(_spans(tensors))
            bucket = (device, _matrix_shape(parameter), parameter.dtype, parameter.grad.dtype)
            rows, keys = buckets.setdefault(bucket, ([], []))
            rows.append(tensors)
            keys.append((update_key(group["sr_seed"], rng_step, index), offset))
        for device_spans in spans.values():
            validate_no_overlap(device_spans)
        # The launches of a device follow each other on its stream, so one workspace serves them all.
        sizes = {}
        for (device, shape, _, _), (rows, _) in buckets.items():
            sizes[device] = max(sizes.get(device, 0), _workspace_bytes(len(rows), *shape))
        workspaces = {d: torch.empty(size, dtype=torch.uint8, device=d) for d, size in sizes.items()}
        for (device, shape, _, _), (rows, keys) in buckets.items():
            _launch(rows, shape, keys, codes, self._hyper(group), ns, workspaces[device])


class MuonHipRN(MuonHip):
    """Muon whose momentum always uses round-to-nearest storage."""

    _forced_rounding = "nearest"

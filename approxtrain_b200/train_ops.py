"""Operators of a Transformer training step around the table products.

=====================  ==================================================================
``residual_norm``      norms before and after a block with its gate and residual scale
``rotary``             rotary positions of queries and keys
``adamw_step``         one AdamW step over many tensors, moments in 32 bits or in 8
=====================  ==================================================================

Same manner as :mod:`approxtrain_b200.ops`, which exports all of them: torch CUDA tensors, one call into ``libamsim.so``
on the current stream, no CPU implementation.  The functions here compute; :mod:`approxtrain_b200.layers` wires the
gradients.
"""
from __future__ import annotations

import array
import contextlib
import ctypes as C
import math

import torch

from ._lib import lib, check, NORM_RMS, NORM_POST, NORM_PRE, NORM_MAX_WIDTH, ROTARY_INTERLEAVED, ROTARY_INVERSE, ROTARY_POS32

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _tensor(t, name: str, like: torch.Tensor = None) -> torch.Tensor:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must live on a CUDA device: there is no CPU implementation")
    if t.dtype not in _TYPES:
        raise TypeError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    if like is not None and t.device != like.device:
        raise ValueError(f"{name} is on {t.device}, expected {like.device}")
    return t


_current_device, _current_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


def _call(device: torch.device, fn, *args) -> None:
    """``fn(current stream, ...)`` with `device` current; raises what the library reports."""
    idx = device.index
    if idx == _current_device():
        check(fn(_current_stream(idx), *args))
    else:
        with torch.cuda.device(idx):
            check(fn(_current_stream(idx), *args))


def _ptr(t):
    return None if t is None else t.data_ptr()


# ---- residual_norm --------------------------------------------------------------------------------
def _norm_pair(pair, name, x):
    """(present, weight, bias) of a norm given as None, (weight, bias) or (None, None)."""
    if pair is None:
        return False, None, None
    w, b = pair
    out = []
    for t, part in ((w, "weight"), (b, "bias")):
        if t is not None:
            t = _tensor(t, f"{name} {part}", x)
            if tuple(t.shape) != (x.shape[-1],):
                raise ValueError(f"{name} {part} must have shape [{x.shape[-1]}], got {list(t.shape)}")
            t = t.contiguous()
        out.append(t)
    return True, out[0], out[1]


def _gate_rows(gate, x) -> int:
    """Rows of the gate: 1 for [width], else the leading axes it shares with x (the rest of them 1)."""
    width = x.shape[-1]
    if gate.dim() == 1 and gate.shape[0] == width:
        return 1
    bad = f"gate must have shape [{width}], x's shape {list(x.shape)}, or that with trailing row axes of 1, got {list(gate.shape)}"
    if gate.dim() != x.dim() or gate.shape[-1] != width:
        raise ValueError(bad)
    rows, shared = 1, True
    for g, n in zip(gate.shape[:-1], x.shape[:-1]):
        shared = shared and g == n
        if shared:
            rows *= g
        elif g != 1:
            raise ValueError(bad)
    return rows


class _NormArgs:
    """Checked arguments of residual_norm, contiguous."""

    def __init__(self, x, block, gate, scale, post, pre, kind, eps):
        x = _tensor(x, "x")
        if x.dim() < 1 or x.shape[-1] < 1:
            raise ValueError(f"x must have at least one column, got shape {list(x.shape)}")
        if x.shape[-1] > NORM_MAX_WIDTH:
            raise ValueError(f"rows of at most {NORM_MAX_WIDTH} elements, got {x.shape[-1]}")
        if kind not in ("layer", "rms"):
            raise ValueError(f"kind must be 'layer' or 'rms', got {kind!r}")
        if not eps >= 0:
            raise ValueError(f"eps must not be negative, got {eps}")
        self.x = x.contiguous()
        self.block = self.gate = None
        if block is not None:
            block = _tensor(block, "block", x)
            if block.shape != x.shape or block.dtype != x.dtype:
                raise ValueError(f"block must match x ({x.dtype}, {list(x.shape)}), got {block.dtype}, {list(block.shape)}")
            self.block = block.contiguous()
        elif post is not None or gate is not None:
            raise ValueError("a norm after the block or a gate needs a block")
        self.gate_rows = 0
        self.width = x.shape[-1]
        self.rows = x.numel() // self.width
        if gate is not None:
            self.gate_rows = _gate_rows(_tensor(gate, "gate", x), x)
            self.gate = gate.contiguous()
        has_post, self.post_w, self.post_b = _norm_pair(post, "post", x)
        has_pre, self.pre_w, self.pre_b = _norm_pair(pre, "pre", x)
        if not has_pre and block is None:
            raise ValueError("neither a block to add nor a norm to take")
        if kind == "rms" and (self.post_b is not None or self.pre_b is not None):
            raise ValueError("rms norms have no bias")
        w_types = {t.dtype for t in (self.post_w, self.post_b, self.pre_w, self.pre_b) if t is not None}
        if len(w_types) > 1:
            raise TypeError(f"weights and biases must have one type, got {sorted(str(t) for t in w_types)}")
        self.w_type = _TYPES[w_types.pop()] if w_types else 0
        self.type = _TYPES[x.dtype]
        self.gate_type = _TYPES[self.gate.dtype] if self.gate is not None else 0
        if self.w_type not in (0, self.type) or self.gate_type not in (0, self.type):
            raise TypeError("weights, biases and gate must be float32 or have x's type")
        self.scale, self.eps = float(scale), float(eps)
        self.pre = has_pre
        self.flags = (NORM_RMS if kind == "rms" else 0) | (NORM_POST if has_post else 0) | (NORM_PRE if has_pre else 0)


def _norm_forward(a: _NormArgs, need_sum: bool, need_stats: bool):
    r = torch.empty_like(a.x) if need_sum or not a.pre else None
    y = torch.empty_like(a.x) if a.pre else None
    stats = torch.empty((a.rows, 4), dtype=torch.float32, device=a.x.device) if need_stats else None
    _call(a.x.device, lib.amsim_residual_norm, a.x.data_ptr(), _ptr(a.block), _ptr(a.gate), _ptr(a.post_w), _ptr(a.post_b),
          _ptr(a.pre_w), _ptr(a.pre_b), _ptr(r), _ptr(y), _ptr(stats), a.rows, a.width, a.gate_rows, a.scale, a.eps, a.type,
          a.w_type, a.gate_type, a.flags)
    return r, y, stats


def residual_norm(x, block=None, gate=None, scale: float = 1.0, post=None, pre=None, kind: str = "layer", eps: float = 1e-3,
                  need_sum: bool = True):
    """The norms around a residual block in one launch:

    ``u = norm(block; post)`` or ``block``; ``r = x + scale * gate * u``; ``y = norm(r; pre)``; returns ``(r, y)``.

    ``post`` (the norm after the block) and ``pre`` (the norm before the next block) are ``(weight, bias)``, either of
    which may be None, or None for no such norm (``y`` is then None).  ``kind``: "layer" norms subtract the mean,
    "rms" norms do not and have no bias.  ``gate``: [width], or x's shape with any number of its trailing row axes 1
    (``[batch, 1, width]``: one per sequence).  x, block: float32, bfloat16 or float16, any leading axes, rows of up to
    32768 elements; weights, biases, gate: float32 or x's type.  Computed in FP32, every output rounded once.
    ``need_sum=False``: ``r`` is not written and returned as None.  For gradients use ``layers.residual_norm``."""
    r, y, _ = _norm_forward(_NormArgs(x, block, gate, scale, post, pre, kind, eps), need_sum, False)
    return r, y


def _norm_backward(dr, dy, x, stats, block=None, gate=None, gate_rows: int = 0, scale: float = 1.0, post_w=None, post_b=None,
                       pre_w=None, pre_b=None, flags: int = NORM_PRE, wants=(True,) * 7):
    """Gradients (x, block, gate, post weight, post bias, pre weight, pre bias) of a checked forward pass from those of its
    outputs (either may be None); ``stats`` is the forward pass's, ``wants`` says which are computed.  The sum is made
    again from x and block, unrounded.  Where x and block are only added (no norm after the block, no gate, scale 1) the block's gradient is x's tensor."""
    like = x
    rows, width = (like.numel() // like.shape[-1], like.shape[-1])
    post, pre = bool(flags & NORM_POST), bool(flags & NORM_PRE)
    device = like.device
    dx = torch.empty_like(like)
    plain = not post and gate is None and scale == 1.0
    dblock = torch.empty_like(like) if wants[1] and not plain else None
    dgate = torch.empty_like(gate) if gate is not None and wants[2] else None

    def grad_of(p, want):
        return torch.empty_like(p) if p is not None and want else None
    dpost_w, dpost_b, dpre_w, dpre_b = (grad_of(p, w) for p, w in zip((post_w, post_b, pre_w, pre_b), wants[3:]))
    weights = next((t for t in (post_w, post_b, pre_w, pre_b) if t is not None), None)
    if dr is None and dy is None:
        for t in (dx, dblock, dgate, dpost_w, dpost_b, dpre_w, dpre_b):
            if t is not None:
                t.zero_()
    else:
        with torch.cuda.device(device) if device.index != _current_device() else contextlib.nullcontext():
            size = lib.amsim_residual_norm_grad_workspace(rows, width, gate is not None, _TYPES[like.dtype], flags)
        ws = torch.empty(size, dtype=torch.uint8, device=device)
        _call(device, lib.amsim_residual_norm_grad, _ptr(dr), _ptr(dy), x.data_ptr(), _ptr(block), _ptr(gate), _ptr(post_w), _ptr(post_b),
              _ptr(pre_w), stats.data_ptr(), dx.data_ptr(), _ptr(dblock), _ptr(dgate), _ptr(dpost_w), _ptr(dpost_b), _ptr(dpre_w),
              _ptr(dpre_b), rows, width, gate_rows, scale, _TYPES[like.dtype], _TYPES[weights.dtype] if weights is not None else 0,
              _TYPES[gate.dtype] if gate is not None else 0, ws.data_ptr() if size else None, size, flags)
    if wants[1] and plain:
        dblock = dx
    return dx, dblock, dgate, dpost_w, dpost_b, dpre_w, dpre_b


# ---- rotary ---------------------------------------------------------------------------------------
class RotaryFrequencies:
    """Angles per position of the rotated pairs (float64, on the device) and the factor on the rotated values."""

    def __init__(self, inv_freq: torch.Tensor, scale: float = 1.0):
        if not isinstance(inv_freq, torch.Tensor) or inv_freq.dtype != torch.float64 or inv_freq.dim() != 1 or inv_freq.numel() == 0:
            raise TypeError("inv_freq must be a float64 tensor of one frequency per pair")
        if not inv_freq.is_cuda:
            raise ValueError("inv_freq must live on a CUDA device: there is no CPU implementation")
        self.inv_freq = inv_freq.contiguous()
        self.scale = float(scale)
        self.rotary_dim = 2 * inv_freq.numel()


def _frequencies64(rotary_dim, base, scaling, factor, original_length, low_turns, high_turns):
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and at least 2, got {rotary_dim}")
    if not base > 0 or not factor > 0:
        raise ValueError("base and factor must be positive")
    i = torch.arange(rotary_dim // 2, dtype=torch.float64)
    if scaling == "base" and rotary_dim > 2:
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    f, scale = base ** (-2.0 * i / rotary_dim), 1.0
    if scaling == "linear":
        f = f / factor
    elif scaling == "blend":
        if not original_length > 0 or not high_turns > low_turns:
            raise ValueError("scaling 'blend' needs original_length > 0 and high_turns > low_turns")
        keep = ((original_length * f / (2 * math.pi) - low_turns) / (high_turns - low_turns)).clamp(0.0, 1.0)
        f = f * keep + f / factor * (1 - keep)
        scale = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    elif scaling not in (None, "base"):
        raise ValueError(f"scaling must be None, 'linear', 'base' or 'blend', got {scaling!r}")
    return f, scale


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling=None, factor: float = 1.0, original_length: int = 0,
                       low_turns: float = 1.0, high_turns: float = 32.0, device="cuda") -> RotaryFrequencies:
    """The frequencies ``base ** (-2 i / rotary_dim)``, scaled for contexts `factor` times as long:

    ``"linear"``  every frequency divided by `factor` (positions interpolated);
    ``"base"``    the base raised by ``factor ** (rotary_dim / (rotary_dim - 2))``, which divides the lowest by `factor`;
    ``"blend"``   frequencies that turn more than `high_turns` times over `original_length` stay, those below `low_turns` are
                  divided by `factor`, linearly between, and rotated values are multiplied by ``0.1 ln(factor) + 1``."""
    f, scale = _frequencies64(rotary_dim, base, scaling, factor, original_length, low_turns, high_turns)
    return RotaryFrequencies(f.to(device), scale)


def _rotary_heads(x, name, like=None):
    x = _tensor(x, name, like)
    if x.dim() not in (3, 4):
        raise ValueError(f"{name} must be [batch, positions, heads, dim] or [positions, heads, dim], got {list(x.shape)}")
    if like is not None and (x.dim() != like.dim() or x.dtype != like.dtype or x.shape[:-2] != like.shape[:-2] or x.shape[-1] != like.shape[-1]):
        raise ValueError(f"{name} must match the first tensor's type, batch, positions and dim, got {x.dtype}, {list(x.shape)}")
    return x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()


def _share_elements(a, b) -> bool:
    """Whether two tensors of one type share an element (True also where that takes long to tell).  A place that both have is a
    solution of: sum of stride x difference of indices = distance between them; found from the longest stride down."""
    if not a.numel() or not b.numel():
        return False
    apart = (b.data_ptr() - a.data_ptr()) // a.element_size()
    if a.is_contiguous() and b.is_contiguous():
        return -b.numel() < apart < a.numel()
    span = {}   # stride -> least and largest difference of indices
    for t, sign in ((a, 1), (b, -1)):
        for n, st in zip(t.shape, t.stride()):
            if n > 1 and st:
                lo, hi = span.get(st, (0, 0))
                span[st] = (lo, hi + n - 1) if sign > 0 else (lo - n + 1, hi)
    strides = sorted(span, reverse=True)
    behind = [(0, 0)]   # what the strides behind each one reach
    for st in strides[:0:-1]:
        behind.insert(0, (behind[0][0] + st * span[st][0], behind[0][1] + st * span[st][1]))
    left = {apart}
    for st, (lo, hi) in zip(strides, behind):
        ranges = [(d, max(span[st][0], -((hi - d) // st)), min(span[st][1], (d - lo) // st)) for d in left]
        if sum(max(0, last - first + 1) for _, first, last in ranges) > 4096:
            return True
        left = {d - st * i for d, first, last in ranges for i in range(first, last + 1)}
    return 0 in left


def _repeats_elements(t) -> bool:
    """Whether an element may have several places in t: where a stride is no longer than all that the shorter ones reach."""
    reach = 0
    for st, n in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n > 1):
        if st <= reach:
            return t.numel() > 0
        reach += st * (n - 1)
    return False


def _strides(x):
    return (0, *x.stride()[:2]) if x.dim() == 3 else x.stride()[:3]


_StrideArray = C.c_longlong * 14


def rotary(q, positions, freqs: RotaryFrequencies, k=None, layout: str = "half", inverse: bool = False, inplace: bool = False):
    """Rotary positions of q (and k): pair i of a head at position p turns by ``p * freqs.inv_freq[i]``.

    q, k: [batch, positions, heads, dim] or [positions, heads, dim], float32, bfloat16 or float16, any strides with a dense
    last axis (``transpose(1, 2)`` of [batch, heads, positions, dim], a slice of a joint projection); k may have other heads
    than q.  ``positions``: int32 or int64, [positions] or [batch, positions].  ``layout``: "half" (pairs half of the rotated
    part apart) or "interleaved" (adjacent).  The first ``freqs.rotary_dim`` elements of a head turn, the rest are
    copied.  ``inverse`` turns back.  ``inplace`` writes over q and k, which must not overlap.  Returns q's result, or both."""
    q = _rotary_heads(q, "q") if not inplace else _tensor(q, "q")
    k_ = None
    if k is not None:
        k_ = _rotary_heads(k, "k", q)
    if inplace:
        for t, name in ((q, "q"), (k, "k")):
            if t is not None and t.shape[-1] != 1 and t.stride(-1) != 1:
                raise ValueError(f"{name} must have a dense last axis to be rotated in place")
            if t is not None and _repeats_elements(t):
                raise ValueError(f"{name} must not be expanded or overlap itself to be rotated in place")
            if t is not None and t.requires_grad and torch.is_grad_enabled():
                raise ValueError(f"{name} requires a gradient: it cannot be rotated in place (layers.rotary keeps gradients)")
        _rotary_heads(q, "q")
        if k is not None and _share_elements(q, k):
            raise ValueError("q and k must not share elements to be rotated in place")
    if not isinstance(freqs, RotaryFrequencies):
        raise TypeError("freqs must be RotaryFrequencies (rotary_frequencies)")
    if freqs.rotary_dim > q.shape[-1]:
        raise ValueError(f"{freqs.rotary_dim} rotated elements in heads of {q.shape[-1]}")
    if layout not in ("half", "interleaved"):
        raise ValueError(f"layout must be 'half' or 'interleaved', got {layout!r}")
    if not isinstance(positions, torch.Tensor) or positions.dtype not in (torch.int32, torch.int64):
        raise TypeError("positions must be an int32 or int64 tensor")
    if positions.device != q.device or freqs.inv_freq.device != q.device:
        raise ValueError(f"positions and frequencies must be on {q.device}")
    batch = q.shape[0] if q.dim() == 4 else 1
    seq = q.shape[-3]
    if tuple(positions.shape) not in ((seq,), (batch, seq)):
        raise ValueError(f"positions must have shape [{seq}] or [{batch}, {seq}], got {list(positions.shape)}")
    out = q if inplace else torch.empty_like(q)
    out2 = (k_ if inplace else torch.empty_like(k_)) if k_ is not None else None
    ps = (0, positions.stride(0)) if positions.dim() == 1 else positions.stride()
    none = (0, 0, 0)
    strides = _StrideArray(*_strides(q), *_strides(out), *(_strides(k_) if k_ is not None else none), *(_strides(out2) if k_ is not None else none), *ps)
    flags = (ROTARY_INTERLEAVED if layout == "interleaved" else 0) | (ROTARY_INVERSE if inverse else 0) | (ROTARY_POS32 if positions.dtype == torch.int32 else 0)
    _call(q.device, lib.amsim_rotary, q.data_ptr(), out.data_ptr(), q.shape[-2], _ptr(k_), _ptr(out2), k_.shape[-2] if k_ is not None else 0,
          positions.data_ptr(), freqs.inv_freq.data_ptr(), batch, seq, q.shape[-1], freqs.rotary_dim, strides, freqs.scale, _TYPES[q.dtype], flags)
    if inplace:  # (a graph that has saved q or k notices)
        torch.autograd.graph.increment_version([q] if k is None else [q, k])
    return out if k is None else (out, out2)


# ---- AdamW ----------------------------------------------------------------------------------------
ADAMW_BLOCK = 256     # elements that share a scale in 8-bit moments
_contiguous, _numel, _device, _data_ptr = torch.Tensor.is_contiguous, torch.Tensor.numel, torch.Tensor.get_device, torch.Tensor.data_ptr


def _address(a: array.array):
    return a.buffer_info()[0]


class AdamWState:
    """Moments and step count of ``adamw_step`` for a list of parameters (float32, bfloat16 or float16, all of one type, on one
    device).

    ``bits=32``: ``exp_avg`` and ``exp_avg_sq``, float32, parameter after parameter.  ``bits=8``: ``exp_avg`` and
    ``exp_avg_sq_root`` (the square root of the second moment) as float8_e4m3fn, every parameter padded to a multiple of
    256 elements, and the scale of every 256 (``exp_avg_scale``, ``exp_avg_sq_scale``): value = code * scale.
    ``moments(i)`` gives those of parameter i in float32.  ``step``: int64 on the device, counted by the steps themselves."""

    def __init__(self, params, bits: int = 32):
        params = list(params)
        if bits not in (8, 32):
            raise ValueError(f"moments of 32 or 8 bits, got {bits}")
        if not params:
            raise ValueError("no parameters")
        for i, p in enumerate(params):
            _tensor(p, f"parameter {i}", params[0])
            if p.dtype != params[0].dtype:
                raise TypeError(f"parameters must have one type, got {p.dtype} beside {params[0].dtype}")
        self.bits, self.device, self.dtype = bits, params[0].device, params[0].dtype
        self.shapes = [tuple(p.shape) for p in params]
        self.sizes = [p.numel() for p in params]
        block = ADAMW_BLOCK if bits == 8 else 1
        self._starts, at = [], 0
        for n in self.sizes:
            self._starts.append(at)
            at += -(-n // block) * block
        kw = dict(device=self.device)
        if bits == 32:
            self.exp_avg, self.exp_avg_sq = (torch.zeros(at, dtype=torch.float32, **kw) for _ in range(2))
            self._moments = ("exp_avg", "exp_avg_sq")
        else:
            self.exp_avg, self.exp_avg_sq_root = (torch.zeros(at, dtype=torch.float8_e4m3fn, **kw) for _ in range(2))
            self.exp_avg_scale, self.exp_avg_sq_scale = (torch.zeros(at // ADAMW_BLOCK, dtype=torch.float32, **kw) for _ in range(2))
            self._moments = ("exp_avg", "exp_avg_scale", "exp_avg_sq_root", "exp_avg_sq_scale")
        self._counter = torch.zeros(2, dtype=torch.int64, **kw)
        self._sizes = array.array("q", self.sizes)

    @property
    def step(self) -> torch.Tensor:
        return self._counter[0]

    def moments(self, i: int):
        """(exp_avg, exp_avg_sq) of parameter i in float32, in its shape."""
        a, n = self._starts[i], self.sizes[i]
        if self.bits == 32:
            m, v = self.exp_avg[a:a + n], self.exp_avg_sq[a:a + n]
        else:
            b = slice(a // ADAMW_BLOCK, -(-(a + n) // ADAMW_BLOCK))
            codes = slice(b.start * ADAMW_BLOCK, b.stop * ADAMW_BLOCK)
            m = (self.exp_avg[codes].float().view(-1, ADAMW_BLOCK) * self.exp_avg_scale[b, None]).view(-1)[:n]
            v = (self.exp_avg_sq_root[codes].float().view(-1, ADAMW_BLOCK) * self.exp_avg_sq_scale[b, None]).square().view(-1)[:n]
        return m.view(self.shapes[i]), v.view(self.shapes[i])

    def state_dict(self) -> dict:
        return {"bits": self.bits, "shapes": list(self.shapes), "step": self.step.clone(), **{k: getattr(self, k).clone() for k in self._moments}}

    def load_state_dict(self, state: dict) -> None:
        """Takes over what ``state_dict`` gave; a state that does not fit is refused and nothing is changed."""
        if state["bits"] != self.bits or [tuple(s) for s in state["shapes"]] != self.shapes:
            raise ValueError("the state is of other parameters or other bits")
        step = int(state["step"])
        for k in self._moments:
            if state[k].shape != getattr(self, k).shape or state[k].dtype != getattr(self, k).dtype:
                raise ValueError(f"{k} does not match")
        with torch.no_grad():
            self._counter[0] = step
            for k in self._moments:
                getattr(self, k).copy_(state[k])


def _rate(value, name, device):
    """(number, address of a number on the device)."""
    if not isinstance(value, torch.Tensor):
        return float(value), None
    if value.dtype != torch.float32 or value.numel() != 1 or value.device != device:
        raise ValueError(f"{name} must be a number or a float32 tensor of one element on {device}")
    return 1.0, value.data_ptr()


def adamw_step(params, grads, state: AdamWState, lr, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay=0.0, grad_scale=1.0, seed: int = 0) -> None:
    """One AdamW step (weight decay beside the gradient) over `params`, in place, with the moments and the step count in
    `state`; in FP32 whatever the types, two launches at most up to 1280 tensors.

    ``p -= lr * weight_decay * p``; ``m = b1 m + (1 - b1) g``; ``v = b2 v + (1 - b2) g^2``;
    ``p -= lr / (1 - b1^t) * m / (sqrt(v / (1 - b2^t)) + eps)``, g = grad * grad_scale.

    `params`, `grads`: lists in the order of the state, dense, of any alignment; gradients have the parameters' type or
    are float32.  `weight_decay`: a number, or one per parameter.  `lr`, `grad_scale`: numbers, or float32 tensors of
    one element on the device (read when the step runs, so a captured step follows them).  `seed`: of the random rounding
    of 8-bit moments.  Gradients have to be finite: one that is not makes its block's moments and its parameter so."""
    if not isinstance(state, AdamWState):
        raise TypeError("state must be an AdamWState")
    n = len(state.sizes)
    for ts, name in ((params, "params"), (grads, "grads")):
        if len(ts) != n:
            raise ValueError(f"{n} {name} expected, got {len(ts)}")
        if list(map(_numel, ts)) != state.sizes:
            raise ValueError(f"the sizes of {name} are not those of the state's parameters")
        if not all(map(_contiguous, ts)):
            raise ValueError(f"{name} must be contiguous")
        if set(map(_device, ts)) != {state.device.index}:
            raise ValueError(f"{name} must be on {state.device}")
    types = {t.dtype for t in grads}
    if {t.dtype for t in params} != {state.dtype} or len(types) != 1 or not types <= {state.dtype, torch.float32}:
        raise TypeError(f"params must be {state.dtype}, grads all {state.dtype} or all float32")
    if isinstance(weight_decay, (int, float)):
        decay = array.array("f", (weight_decay,)) * n
    else:
        decay = array.array("f", weight_decay)
        if len(decay) != n:
            raise ValueError(f"weight_decay: a number or {n} of them, got {len(decay)}")
    b1, b2 = betas
    if not (0 <= b1 < 1 and 0 <= b2 < 1) or not eps >= 0:
        raise ValueError(f"betas in [0, 1) and eps >= 0 expected, got {betas}, {eps}")
    lr, lr_at = _rate(lr, "lr", state.device)
    scale, scale_at = _rate(grad_scale, "grad_scale", state.device)
    p_at, g_at = array.array("Q", map(_data_ptr, params)), array.array("Q", map(_data_ptr, grads))
    if len(set(p_at)) < n and len({a for a, k in zip(p_at, state.sizes) if k}) < sum(map(bool, state.sizes)):
        raise ValueError("a parameter is listed twice (tied weights are updated once)")
    if state.bits == 32:
        m, ms, v, vs = state.exp_avg.data_ptr(), None, state.exp_avg_sq.data_ptr(), None
    else:
        m, ms, v, vs = (getattr(state, k).data_ptr() for k in state._moments)
    _call(state.device, lib.amsim_adamw, n, _address(p_at), _address(g_at), _address(state._sizes), _address(decay), m, ms, v, vs,
          state._counter.data_ptr(), lr, lr_at, b1, b2, eps, scale, scale_at, seed & 0xFFFFFFFF, _TYPES[state.dtype], _TYPES[types.pop()], state.bits)
    torch.autograd.graph.increment_version(params)  # (a graph that has saved a parameter notices)

"""AdamW over many tensors at once on librst (``rst_adamw_*``, include/rst.h), beside the trainers' RMSprop
(``styleTransferTrainingModel.RMSprop``, train_network.py:102).

One launch steps every variable, whatever their number and sizes; with ``global_clipnorm`` one more launch forms the
gradient's norm over all of them. The moments are kept in 32 bits (8 bytes an element) or in 8 (2 bytes and a scale per
128 elements). ``StyleTransferTrainingModel.compile(optimizer=AdamW(...))`` trains the transfer network and the style
predictor with it; ``build`` takes any float32 device tensors.

The step t, with c = min(1, global_clipnorm / |g|) and t = iterations + 1::

    m = beta_1 m + (1 - beta_1) c g
    v = beta_2 v + (1 - beta_2) (c g)^2
    p -= learning_rate (m / (1 - beta_1^t) / (sqrt(v / (1 - beta_2^t)) + epsilon) + weight_decay p)
"""
from __future__ import annotations

import ctypes
import math
import weakref
from typing import List, Optional, Sequence, Tuple, Union

import torch

from . import _lib

BLOCK = 128          # elements of one 8-bit state block
_DTYPES = {torch.float32: _lib.DTYPES["float32"], torch.bfloat16: _lib.DTYPES["bfloat16"]}


class AdamW:
    """``weight_decay`` applies to the variables ``build`` was given ``decay`` for (by default those with more than one
    dimension: kernels, not biases and norm scales). ``global_clipnorm``: scale the gradients so that their joint norm
    is at most this; a step whose norm is not finite then changes nothing. ``state_bits``: 32 or 8. ``seed``: of the
    random rounding of 8-bit second moments (reproducible: a hash of element, step and seed). ``learning_rate``,
    ``weight_decay`` and ``epsilon`` are finite in 32 bits, ``epsilon`` is at least 2^-126.

    The hyperparameters are attributes and may be changed between steps. A step captured into a graph keeps those it was
    captured with, and counts on with every replay (the step count is on the device); keep the optimizer while the graph
    replays. One step of an optimizer at a time: not on two streams at once."""

    def __init__(self, learning_rate: float = 1e-3, weight_decay: float = 4e-3, beta_1: float = 0.9,
                 beta_2: float = 0.999, epsilon: float = 1e-7, global_clipnorm: Optional[float] = None,
                 state_bits: int = 32, seed: int = 0):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits!r}")
        if global_clipnorm is not None and not global_clipnorm > 0.0:
            raise ValueError(f"global_clipnorm must be positive and finite, or None, got {global_clipnorm!r}")
        self.learning_rate, self.weight_decay = float(learning_rate), float(weight_decay)
        self.beta_1, self.beta_2, self.epsilon = float(beta_1), float(beta_2), float(epsilon)
        self.global_clipnorm = None if global_clipnorm is None else float(global_clipnorm)
        self.state_bits, self.seed = int(state_bits), int(seed)
        self._handle = self._owner = None
        self._config, self._config_of = _lib.RstAdamwConfig(), None
        self._check_config()

    def __del__(self):
        try:
            if getattr(self, '_handle', None) is not None:
                _lib.load().rst_adamw_destroy(self._handle)
                self._handle = None
        except Exception:
            pass

    def _check_config(self):
        clip = self.global_clipnorm
        of = (self.learning_rate, self.weight_decay, self.beta_1, self.beta_2, self.epsilon, clip, self.seed)
        if of == self._config_of:
            return self._config
        c = _lib.RstAdamwConfig()
        c.learning_rate, c.weight_decay, c.epsilon = self.learning_rate, self.weight_decay, self.epsilon
        c.beta_1, c.beta_2, c.seed = self.beta_1, self.beta_2, self.seed & 0xFFFFFFFF
        c.global_clipnorm = 0.0 if clip is None else clip
        if not (0.0 <= c.beta_1 < 1.0 and 0.0 <= c.beta_2 < 1.0):
            raise ValueError(f"beta_1 and beta_2 must lie in [0, 1), got {c.beta_1} and {c.beta_2}")
        rate, decay, epsilon = (ctypes.c_float(x).value for x in (c.learning_rate, c.weight_decay, c.epsilon))
        if not (math.isfinite(rate) and math.isfinite(decay) and 2.0 ** -126 <= epsilon < math.inf):
            raise ValueError("learning_rate, weight_decay and epsilon must be finite in 32 bits, epsilon at least 2^-126, "
                             f"got {c.learning_rate}, {c.weight_decay} and {c.epsilon}")
        if not 0.0 <= c.global_clipnorm < math.inf:
            raise ValueError(f"global_clipnorm must be positive and finite, or None, got {clip!r}")
        self._config, self._config_of = c, of
        return c

    # ------------------------------------------------------------------ state
    def build(self, variables: Sequence[torch.Tensor], decay: Optional[Sequence[bool]] = None):
        """Bind the variables (contiguous float32 tensors of one device, updated in place) and make their states, zeros.
        The gradient bucket holds the variables' gradients one after the other, in this order. The memory that a
        variable has now is what the steps update: one whose ``data`` is replaced later is not followed."""
        variables = list(variables)
        if not variables:
            raise ValueError("no variables")
        device = variables[0].device
        for v in variables:
            _lib.dev_ptr(v)
            if v.device != device:
                raise ValueError(f"variables are on {device} and {v.device}")
        if decay is None:
            decay = [v.dim() > 1 for v in variables]
        counts = [v.numel() for v in variables]
        self._build([v.data_ptr() for v in variables], counts, None, decay, device)
        self._variables = [v.detach() for v in variables]       # keeps that memory, and shares its version
        bases = [v if v._base is None else v._base for v in variables]
        self._versioned = list({id(b): v for b, v in zip(bases, self._variables)}.values())   # (a buffer's views have one)

    def _build(self, pointers: Sequence[int], counts: Sequence[int], offsets: Optional[Sequence[int]],
               decay: Sequence[bool], device, owner=None):
        """``offsets``: each variable's first element in the gradient bucket (None: no gaps). ``owner``: the object that
        owns the variables' memory where that is no tensor."""
        if self._handle is not None:
            raise ValueError("this optimizer already has variables: use one AdamW for each model")
        if len(decay) != len(counts):
            raise ValueError(f"{len(counts)} variables, but decay for {len(decay)}")
        if not any(counts):
            raise ValueError("no variable has an element")
        spans = sorted((p, p + 4 * n) for p, n in zip(pointers, counts) if n)
        if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
            raise ValueError("two variables share memory")
        if offsets is None:
            offsets, at = [], 0
            for n in counts:
                offsets.append(at)
                at += n
        self._counts = list(counts)
        self._bucket_size = max((o + n for o, n in zip(offsets, counts)), default=0)
        n, blocks = sum(counts), sum((c + BLOCK - 1) // BLOCK for c in counts)
        self.device = torch.device(device)
        self._index = self.device.index if self.device.index is not None else torch.cuda.current_device()
        with torch.cuda.device(self.device):
            if self.state_bits == 32:
                self.m, self.v = torch.zeros(n, device=device), torch.zeros(n, device=device)
                self.m_scale = self.v_scale = None
            else:
                self.m, self.v = (torch.zeros(blocks, BLOCK, dtype=torch.uint8, device=device)
                                  .view(torch.float8_e4m3fn) for _ in range(2))
                self.m_scale, self.v_scale = torch.zeros(blocks, device=device), torch.zeros(blocks, device=device)
            self._iterations = torch.zeros(1, dtype=torch.int64, device=device)
            self.global_norm = torch.zeros((), device=device)
            table = (_lib.RstAdamwTensor * len(counts))(*zip(pointers, counts, offsets, map(bool, decay)))
            scales = (0, 0) if self.state_bits == 32 else (self.m_scale.data_ptr(), self.v_scale.data_ptr())
            state = _lib.RstAdamwState(self.m.data_ptr(), self.v.data_ptr(), *scales, self._iterations.data_ptr(),
                                       self.global_norm.data_ptr())
            h = ctypes.c_void_p()
            _lib.check(_lib.load().rst_adamw_create(table, len(counts), self.state_bits, ctypes.byref(state),
                                                    ctypes.byref(h)))
        self._handle = h
        self._memory = (self.m, self.v, self.m_scale, self.v_scale, self._iterations, self.global_norm)   # the handle's
        self._variables, self._versioned = None, []
        self._owner = None if owner is None else weakref.ref(owner)

    def _require_built(self):
        if self._handle is None:
            raise ValueError("the optimizer has no variables yet: build() it, or compile a training model with it")
        if self._owner is not None and self._owner() is None:
            raise ValueError("the model whose variables this optimizer steps no longer exists")

    def _bound_to(self, owner) -> bool:
        return self._handle is not None and self._owner is not None and self._owner() is owner

    @property
    def iterations(self) -> int:
        """Steps taken (reads the device)."""
        self._require_built()
        return int(self._iterations.item())

    @iterations.setter
    def iterations(self, value: int):
        self._require_built()
        if value < 0:
            raise ValueError("iterations must not be negative")
        self._iterations.fill_(int(value))

    def slots(self) -> Tuple[List[torch.Tensor], List[torch.Tensor]]:
        """The moments m and v of every variable as flat float32 tensors (8-bit states: the values they stand for, at most
        float32's largest number)."""
        self._require_built()
        out, top = [], torch.finfo(torch.float32).max
        for s, scale in ((self.m, self.m_scale), (self.v, self.v_scale)):
            if self.state_bits == 32:
                out.append([t.clone() for t in s.split(self._counts)])
            else:
                flat = (s.float() * scale[:, None]).clamp_(-top, top).reshape(-1)      # (a NaN stays)
                rows = [BLOCK * ((c + BLOCK - 1) // BLOCK) for c in self._counts]
                out.append([t[:c].clone() for t, c in zip(flat.split(rows), self._counts)])
        return out[0], out[1]

    def set_slots(self, m: Sequence[torch.Tensor], v: Sequence[torch.Tensor]):
        """Restore the moments (one tensor per variable, any shape of its size). 8-bit states round to nearest, with the
        scale max / 448 of each block."""
        self._require_built()
        rows = []
        for values in (m, v):
            rows.append([torch.as_tensor(t, dtype=torch.float32, device=self.device).reshape(-1) for t in values])
            if [t.numel() for t in rows[-1]] != self._counts:
                raise ValueError("slots do not match the variables")
        for values, s, scale in zip(rows, (self.m, self.v), (self.m_scale, self.v_scale)):
            if self.state_bits == 32:
                s.copy_(torch.cat(values))
                continue
            x = torch.cat([torch.nn.functional.pad(t, (0, -t.numel() % BLOCK)) for t in values]).view(-1, BLOCK).double()
            finite = x.isfinite()                              # (the others: a NaN code, and no part in the scale)
            largest = (torch.where(finite, x.abs(), 0.0).amax(1) / 448.0).float()
            scale.copy_(torch.where(largest < 2.0 ** -126, 0.0, largest))
            some = (scale > 0)[:, None]
            y = torch.where(some, x / torch.where(some, scale[:, None].double(), 1.0), 0.0).float().clamp(-448.0, 448.0)
            if s is self.v:                  # above zero stays above zero: the step divides by its root
                y = torch.where((x > 0) & some, y.clamp(min=2.0 ** -9), y)
            s.copy_(torch.where(finite, y, float('nan')).to(torch.float8_e4m3fn))

    # ------------------------------------------------------------------ step
    def apply_gradients(self, gradients: Union[torch.Tensor, Sequence[torch.Tensor]]):
        """One step on the current stream. ``gradients``: the bucket (one contiguous tensor, float32 or bfloat16), or a
        list of one contiguous tensor per variable, all of one dtype. Autograd sees the variables change, as in any other
        operation in place (a captured step: when it is captured, not when it replays)."""
        self._require_built()
        if self._owner is not None:
            raise ValueError("these variables are a training model's, whose train_step steps them")
        self._apply(gradients)
        torch.autograd.graph.increment_version(self._versioned)

    def _apply(self, gradients):
        if torch.cuda.current_device() != self._index:
            with torch.cuda.device(self.device):
                return self._apply(gradients)
        lib, config, stream = _lib.load(), self._check_config(), _lib.device_stream(self._index)
        if isinstance(gradients, torch.Tensor):
            if gradients.numel() != self._bucket_size:
                raise ValueError(f"the gradient bucket must have {self._bucket_size} elements, got {gradients.numel()}")
            pointer, dtype = self._gradient(gradients)
            _lib.check(lib.rst_adamw_step(self._handle, pointer, dtype, ctypes.byref(config), stream))
        else:
            gradients = list(gradients)
            if [-1 if g is None else g.numel() for g in gradients] != self._counts:
                raise ValueError("one gradient of its variable's size is needed for every variable")
            rows = [self._gradient(g) for g in gradients]
            dtype = rows[0][1]
            if any(d != dtype for _, d in rows):
                raise ValueError("gradients must all be float32 or all bfloat16")
            pointers = (ctypes.c_void_p * len(rows))(*[p for p, _ in rows])
            _lib.check(lib.rst_adamw_step_tensors(self._handle, pointers, len(rows), dtype, ctypes.byref(config), stream))

    def _gradient(self, g: torch.Tensor) -> Tuple[int, int]:
        if g.device != self.device:
            raise ValueError(f"gradients must be on {self.device}, got {g.device}")
        if g.dtype not in _DTYPES:
            raise ValueError(f"gradients must be float32 or bfloat16, got {g.dtype}")
        if not g.is_contiguous():
            raise ValueError("gradients must be contiguous")
        return g.data_ptr(), _DTYPES[g.dtype]


__all__ = ['AdamW', 'BLOCK']

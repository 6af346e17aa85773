"""``AdamW`` over a model's weights: one launch per step for the whole list of tensors (``csrc/adamw.cu``), first and second
moments in 32 or in 8 bits.

    weights = {name: w.cuda() for name, w in init_weights(spec, seed).items()}
    optimiser = AdamW(weights, lr=1e-3, state_bits=8, rounding="random")
    optimiser.step(gradients)                       # {name: gradient}; tensors without one stay as they are

With t the number of the step:

    m = beta1 m + (1 - beta1) g        v = beta2 v + (1 - beta2) g^2
    p = p (1 - lr weight_decay) - lr / (1 - beta1^t) m / (sqrt(v) / sqrt(1 - beta2^t) + eps)

Weights and arithmetic are float32; gradients float32, bfloat16 or float16; ``copies`` are optional bfloat16 or float16
tensors that a step leaves with the new weights (for products in 16 bits). With ``state_bits=8`` each 256 values of a tensor
share a scale s per moment, the largest of them / 448: m is held as e4m3(m / s), v as e4m3(sqrt(v) / s), never as zero
where v is not. A gradient that is not finite makes the moments of its value (with 8 bits: of its 256 values) not finite, and
with them the weights.

Moments in 8 bits are rounded to the nearest or, with ``rounding="random"``, v at random (m always to the nearest). To the nearest each
step is the best it can be, but v does not follow its moving average over many: what a step changes, 0.05 % of the root with beta2 =
0.999, is less than half of the 6 to 12 % between two codes, so a value keeps its ratio to the largest of its 256. Where the sizes of
gradients change while weights are trained, that is off by factors: at 3,000 steps after all sizes were drawn anew, from lognormals
of e^0.5, the roots of 90 % of the values were 0.3 to 1.8 of the true ones and updates twice as large; of values whose gradients fell to
a tenth many stayed 9 times too large. At random the expected v is the one of 32 bits at every step, and roots are 0.71 to 1.32 of the true
ones (90 %) in both cases. So: ``rounding="random"`` for runs of more than a few hundred steps. The random bits are those of ``seed``, the
number of the step and the place of the value: runs repeat bit by bit, also captured or continued from loaded moments.

The list of tensors and where they lie are those of the construction; gradients share no memory with weights, copies or moments.
Steps of one optimiser follow one another: not two at once on two streams. A step runs on the current stream of the weights' device,
allocates nothing and can be captured: the number of the step is counted on the device, the learning rate and the other constants are
those at capture. There is no CPU path.
"""

from __future__ import annotations

import ctypes
import math
import operator

import numpy as np
import torch

from . import _lib
from .grouped import TYPES, _launch

BLOCK = _lib.ADAMW_BLOCK
_place, _type = torch.Tensor.data_ptr, operator.attrgetter("dtype")


def _share_memory(tensors) -> bool:
    """Whether two of these contiguous tensors overlap."""
    held = sorted((t.data_ptr(), t.numel() * t.element_size()) for t in tensors if t.numel())
    return any(here + size > there for (here, size), (there, _) in zip(held, held[1:]))


class AdamW:
    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.01,
                 state_bits: int = 32, copies=None, rounding: str = "nearest", seed: int = 0):
        self.names = list(params) if isinstance(params, dict) else list(range(len(params)))
        self.params = [params[k] for k in self.names]
        if not self.params:
            raise ValueError("AdamW: no tensors")
        if state_bits not in (8, 32):
            raise ValueError("AdamW: state_bits is 8 or 32")
        if rounding not in ("nearest", "random") or (rounding == "random" and state_bits != 8):
            raise ValueError("AdamW: rounding is 'nearest' or, with state_bits=8, 'random'")
        if not 0 <= int(seed) < 2 ** 31 - 1:
            raise ValueError("AdamW: seed is a number from 0 to 2^31 - 2")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
            raise ValueError("AdamW: betas in [0, 1)")
        if not all(0.0 <= x < math.inf for x in (lr, eps, weight_decay)):
            raise ValueError("AdamW: lr, eps and weight_decay must be finite and not negative")
        self.lr, self.betas, self.eps, self.weight_decay = float(lr), tuple(float(b) for b in betas), float(eps), float(weight_decay)
        self.state_bits = int(state_bits)
        self.rounding, self.seed = rounding, int(seed)
        self.device = self.params[0].device
        for p in self.params:
            if not p.is_cuda:
                raise ValueError("AdamW: the weights must be CUDA tensors, there is no CPU path")
            if p.dtype != torch.float32 or not p.is_contiguous() or p.device != self.device:
                raise ValueError("AdamW: the weights must be contiguous float32 tensors on one device")
        if isinstance(copies, dict):
            if set(copies) - set(self.names):
                raise ValueError(f"AdamW: copies of unknown tensors: {sorted(map(str, set(copies) - set(self.names)))}")
            copies = [copies.get(k) for k in self.names]
        elif copies is not None and len(copies) != len(self.params):
            raise ValueError(f"AdamW: {len(copies)} copies for {len(self.params)} tensors")
        self.copies = [None] * len(self.params) if copies is None else list(copies)
        self._copy_type = 0
        for p, c in zip(self.params, self.copies):
            if c is None:
                continue
            if c.dtype not in (torch.bfloat16, torch.float16) or not c.is_contiguous() or c.device != self.device or c.shape != p.shape:
                raise ValueError("AdamW: a copy must be a contiguous bfloat16 or float16 tensor of its weights' shape")
            if self._copy_type not in (0, TYPES[c.dtype]):
                raise ValueError("AdamW: the copies must have one type")
            self._copy_type = TYPES[c.dtype]
        if _share_memory([t for t in (*self.params, *self.copies) if t is not None]):
            raise ValueError("AdamW: a tensor is listed twice, or two share memory")
        # where weights and copies lie, and what keeps that memory while the optimiser lives
        self._listed = [t for t in (*self.params, *self.copies) if t is not None]
        self._places, self._held = [t.data_ptr() for t in self._listed], [t.detach() for t in self._listed]
        # what a step writes to, for autograd, of each tensor (inference tensors have no version to count)
        self._written = [[t for t in pair if t is not None and not t.is_inference()] for pair in zip(self.params, self.copies)]
        self._all_written = sum(self._written, [])
        self.lib = _lib.load()
        self.blocks, blocks = [], 0
        for p in self.params:
            self.blocks.append(blocks)
            blocks += -(-p.numel() // BLOCK)
        blocks = max(1, blocks)                          # (a list of empty tensors has somewhere to point to as well)
        held = torch.float32 if self.state_bits == 32 else torch.float8_e4m3fn
        with torch.cuda.device(self.device):
            # first moments, and second moments (their square roots in 8 bits), each tensor from the start of a block
            self.m = torch.zeros(blocks * BLOCK, dtype=torch.float32, device=self.device).to(held)
            self.v = torch.zeros(blocks * BLOCK, dtype=torch.float32, device=self.device).to(held)
            scale = lambda: torch.full((blocks,), 2.0 ** -126, device=self.device) if self.state_bits == 8 else None  # noqa: E731
            self.m_scale, self.v_scale = scale(), scale()
            self._state = torch.tensor([0.0, 1.0, 1.0, 0.0], dtype=torch.float64, device=self.device)
        self._shapes, self._index = [p.shape for p in self.params], self.device.index
        self._tensors = (_lib.AdamwTensorStruct * len(self.params))()
        for k, p in enumerate(self.params):
            t = self._tensors[k]
            t.p, t.values, t.block = p.data_ptr(), p.numel(), self.blocks[k]
            t.copy = None if self.copies[k] is None else self.copies[k].data_ptr()
        # the gradients' pointers of the list above, as one column
        self._pointers = np.frombuffer(self._tensors, dtype=np.int64).reshape(len(self.params), -1)[:, 1]
        self._args = _lib.AdamwStruct()
        # whether a step has been captured, and the moments that captured steps go on with since others were loaded
        self._captured, self._replaced = False, []

    def _fill_args(self) -> None:
        a = self._args
        a.moment_bits, a.copy_type = self.state_bits, self._copy_type
        a.random = 1 + self.seed if self.rounding == "random" else 0
        a.lr, a.beta1, a.beta2, a.eps, a.weight_decay = self.lr, *self.betas, self.eps, self.weight_decay
        a.m, a.v, a.state = self.m.data_ptr(), self.v.data_ptr(), self._state.data_ptr()
        if self.state_bits == 8:
            a.m_scale, a.v_scale = self.m_scale.data_ptr(), self.v_scale.data_ptr()

    def step(self, grads) -> None:
        """One step along ``grads`` (a dictionary or sequence like the weights; a missing or ``None`` gradient leaves its
        tensor and its moments as they are). Counts as a step if any tensor that has values has a gradient."""
        if isinstance(grads, dict):
            unknown = set(grads) - set(self.names)
            if unknown:
                raise ValueError(f"AdamW.step: gradients of unknown tensors: {sorted(map(str, unknown))}")
            grads = [grads.get(k) for k in self.names]
        elif len(grads) != len(self.params):
            raise ValueError(f"AdamW.step: {len(grads)} gradients for {len(self.params)} tensors")
        # (mapped methods: looking over 117 small tensors takes the host longer than their step takes the device, 17 us)
        if list(map(_place, self._listed)) != self._places:
            raise ValueError("AdamW.step: a tensor of the list has been given other memory since")
        shapes, written = self._shapes, self._all_written
        try:
            self._pointers[:] = list(map(_place, grads))
        except TypeError:                                # a gradient is None
            self._pointers[:] = [0 if g is None else g.data_ptr() for g in grads]
            written = sum((w for w, g in zip(self._written, grads) if g is not None), [])
            shapes = [s for s, g in zip(shapes, grads) if g is not None]
            grads = [g for g in grads if g is not None]
            if not grads:
                return
        kinds = set(map(_type, grads))
        if len(kinds) != 1 or not kinds <= set(TYPES):
            raise ValueError("AdamW.step: the gradients must have one type, float32, bfloat16 or float16")
        if [g.shape for g in grads] != shapes or not all(map(torch.Tensor.is_contiguous, grads)) or \
                set(map(torch.Tensor.get_device, grads)) != {self._index}:
            raise ValueError("AdamW.step: a gradient must be contiguous, of its weights' shape and on their device")
        self._captured = self._captured or torch.cuda.is_current_stream_capturing()
        self._fill_args()
        self._args.grad_type = TYPES[kinds.pop()]
        _lib.check(_launch(self._index, self.lib.fmb_adamw_step, ctypes.byref(self._args), self._tensors, len(self.params)),
                   "fmb_adamw_step")
        # weights and copies have changed in place: a graph that saved one, to go on to its activations, must not run with the new values
        if written:
            torch.autograd.graph.increment_version(written)

    @property
    def steps(self) -> int:
        """Steps done (synchronises)."""
        return int(self._state[0].item())

    def load_moments(self, steps: int, *moments: torch.Tensor) -> None:
        """Continue from the moments of a run of ``steps`` steps: ``m, v`` (32 bits) or ``m, m_scale, v, v_scale`` (8 bits), as
        this class holds them under these names. The optimiser uses the tensors given, it does not copy them; a step captured before
        goes on with the ones it had, which the optimiser keeps for it."""
        names = ("m", "v") if self.state_bits == 32 else ("m", "m_scale", "v", "v_scale")
        if len(moments) != len(names) or int(steps) != steps or steps < 0:
            raise ValueError(f"AdamW.load_moments: steps and {', '.join(names)}")
        for name, t in zip(names, moments):
            like = getattr(self, name)
            if t.shape != like.shape or t.dtype != like.dtype or t.device != like.device or not t.is_contiguous():
                raise ValueError(f"AdamW.load_moments: {name} must be a contiguous {like.dtype} tensor {tuple(like.shape)}")
            if t.data_ptr() % 16:
                raise ValueError(f"AdamW.load_moments: {name} must start at a multiple of 16 bytes")
        if _share_memory([*moments, *self._listed]):
            raise ValueError("AdamW.load_moments: two of the moments share memory, or one with a weight or copy")
        if self._captured:
            self._replaced.extend(getattr(self, name) for name in names)
        for name, t in zip(names, moments):
            setattr(self, name, t)
        self._state.copy_(torch.tensor([steps, self.betas[0] ** steps, self.betas[1] ** steps, 0.0], dtype=torch.float64))

    def moments(self, name) -> tuple[torch.Tensor, torch.Tensor]:
        """First and second moments of one tensor in float32, in its shape."""
        k = self.names.index(name)
        p, b = self.params[k], self.blocks[k]
        n = -(-p.numel() // BLOCK)
        m, v = (t[b * BLOCK:(b + n) * BLOCK].float().view(n, BLOCK) for t in (self.m, self.v))
        if self.state_bits == 8:
            m, v = m * self.m_scale[b:b + n, None], (v * self.v_scale[b:b + n, None]) ** 2
        return tuple(t.reshape(-1)[:p.numel()].view(p.shape).clone() for t in (m, v))


__all__ = ["AdamW", "BLOCK"]

"""AdamW over many tensors where they are (`tv_adamw_*`, `csrc/adamw.hip`).

The reference trains with tensorkit's RMSprop / Adam over the model's parameters (`train.py:417-426`);
`train.FlatOptimizer` is that update over one flat fp32 buffer.  `AdamW` is for parameters that are
not in such a buffer, or not in fp32: decoupled weight decay per tensor, clipping by the global norm,
16-bit parameters with an fp32 master, and moments in 32 bits or in 8 bits with one scale per block.
"""
import ctypes
from typing import Dict, Iterable, Optional, Sequence, Union

import torch

from . import hip

__all__ = ['AdamW']

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}      # TV_DTYPE_*
BLOCK = 256                                                            # TV_ADAMW_BLOCK


class AdamW(object):
    """One AdamW step over all of `params` per `step()`: three launches with clipping, two without,
    one for few tensors without clipping and guard (one or two more for every 384 tensors).

        m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2
        p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)

    * `params`: contiguous fp32 / bf16 / fp16 tensors on one GPU, none overlapping another.  16-bit
      parameters are rounded copies of an fp32 master in `state['master']`; an element that somebody
      else wrote (a loaded checkpoint) is taken over by the master in the next step.
    * `weight_decay`: one number, or one per parameter.
    * `state_bits` 32: `state['exp_avg']`, `state['exp_avg_sq']` in fp32.  8: `state['exp_avg8']` and
      `state['exp_rms8']` (torch.float8_e4m3fn; sqrt(v), not v) in units of `state['exp_avg_scale']` /
      `state['exp_rms_scale']`, one fp32 scale per 256 elements; rounded stochastically by a hash of
      (the low 32 bits of `seed`, step, element), so a run is reproducible bit for bit.
    * all state buffers are flat: tensor i begins at `offsets[i]`, a multiple of 256.
    * the step counter and the learning rate are on the device: `step()` never waits for the GPU and
      may be captured into a graph (capture after the first eager step; `set_lr` between replays is
      seen by them).  A replay updates the parameters where they were when it was captured, and needs
      the optimizer to be alive.  A tensor whose gradient is None is left as it is, state included; the
      step counter is one for all tensors.
    * calls on one optimizer must be ordered: one stream, or events between them.
    """

    def __init__(self, params: Iterable[torch.Tensor], lr: float = 1e-3, betas=(0.9, 0.999),
                 eps: float = 1e-8, weight_decay: Union[float, Sequence[float]] = 0.01,
                 state_bits: int = 32, seed: int = 0):
        self.params = list(params)
        if not self.params:
            raise ValueError('AdamW needs at least one parameter')
        if state_bits not in (8, 32):
            raise ValueError(f'state_bits must be 8 or 32, got {state_bits}')
        n = len(self.params)
        decay = [float(weight_decay)] * n if isinstance(weight_decay, (int, float)) \
            else [float(d) for d in weight_decay]
        if len(decay) != n:
            raise ValueError(f'{len(decay)} weight decays for {n} parameters')
        self.device = self.params[0].device
        for i, p in enumerate(self.params):
            if not p.is_cuda:
                raise hip.HipLibraryError(
                    f'parameter {i} is on {p.device}: the accelerated path runs on the GPU only '
                    f'(there is no CPU fallback)')
            if p.device != self.device:
                raise ValueError(f'parameter {i} is on {p.device}, the first one on {self.device}')
            if p.dtype not in _DTYPES:
                raise TypeError(f'parameter {i} must be float32, bfloat16 or float16, got {p.dtype}')
            if not p.is_contiguous() or p.is_neg():
                raise ValueError(f'parameter {i} must be contiguous (and no negated view)')
        self.state_bits, self.seed = state_bits, int(seed)
        self.betas, self.eps, self.lr = (float(betas[0]), float(betas[1])), float(eps), float(lr)
        self._captured_lr = False
        self.weight_decay = decay
        self._make_arrays()
        lib = hip.lib()
        total = int(lib.tv_adamw_state_elements(n, self._sizes))
        self.offsets, at = [], 0
        for p in self.params:
            self.offsets.append(at)
            at += (p.numel() + BLOCK - 1) // BLOCK * BLOCK
        assert at == total

        def zeros(count, dtype=torch.float32):
            return torch.zeros(count, dtype=dtype, device=self.device)

        self._state: Dict[str, torch.Tensor] = {}
        if state_bits == 32:
            self._state.update(exp_avg=zeros(total), exp_avg_sq=zeros(total))
        else:
            for name in ('exp_avg', 'exp_rms'):
                self._state[name + '8'] = zeros(total, torch.uint8).view(torch.float8_e4m3fn)
                self._state[name + '_scale'] = zeros(total // BLOCK)
        if any(p.dtype != torch.float32 for p in self.params):
            self._state['master'] = zeros(total)
            for at, p in zip(self.offsets, self.params):
                self._state['master'][at:at + p.numel()].copy_(p.detach().reshape(-1))
        self._control = zeros(int(lib.tv_adamw_control_bytes()) // 8, torch.int64)
        self._write_control(0)
        self._workspace = zeros(int(lib.tv_adamw_workspace_bytes(n)) // 8, torch.float64)
        self.grad_norm = torch.zeros((), dtype=torch.float64, device=self.device)
        self._start()

    # -- set-up ------------------------------------------------------------------------
    def _make_arrays(self) -> None:
        n = len(self.params)
        self._sizes = hip.array_type(ctypes.c_int64, n)(*[p.numel() for p in self.params])
        self._dtypes = hip.array_type(ctypes.c_int, n)(*[_DTYPES[p.dtype] for p in self.params])
        self._decay = hip.array_type(ctypes.c_double, n)(*self.weight_decay)
        self._addresses = hip.array_type(ctypes.c_int64, n)()

    def _start(self) -> None:
        self._lr = self._control.view(torch.float64)[1]
        self._plan = None
        self._captured_plans = []                 # read by every replay of the steps captured with them
        self._make_plan()

    # a copy has addresses of its own: those of its arrays, buffers and parameters, not the original's
    _ADDRESSED = ('_sizes', '_dtypes', '_decay', '_addresses', '_where', '_plan', '_plan_host', '_captured_plans',
                  '_fixed', '_lr')

    def __getstate__(self):
        return {k: v for k, v in self.__dict__.items() if k not in self._ADDRESSED}

    def __setstate__(self, state) -> None:
        self.__dict__.update(state)
        self._make_arrays()
        self._start()

    def _call_host(self, name: str, *args) -> None:
        if getattr(hip.lib(), name)(*args) != 0:
            msg = hip.lib().tv_last_error().decode('utf-8', 'replace')
            raise hip.HipLibraryError(f'{name} failed: {msg}')

    def _write_control(self, step: int) -> None:
        image = torch.zeros(self._control.numel(), dtype=torch.int64)
        self._call_host('tv_adamw_control', int(step), self.lr, self.betas[0], self.betas[1],
                        self.eps, image.data_ptr())
        self._control.copy_(image)

    def _make_plan(self) -> None:
        n = len(self.params)
        where = hip.array_type(ctypes.c_int64, n)(*[p.data_ptr() for p in self.params])
        nbytes = int(hip.lib().tv_adamw_plan_bytes(n, self._sizes))
        image = torch.zeros((nbytes + 7) // 8, dtype=torch.int64)
        self._call_host('tv_adamw_plan', n, self._sizes, self._dtypes,
                        ctypes.addressof(where), self._decay,
                        image.data_ptr(), nbytes)
        if self._plan is not None:
            # a step may still read it, on a stream that is not the one it was allocated on
            self._plan.record_stream(torch.cuda.current_stream(self.device))
        self._plan_host, self._plan, self._where = image, image.to(self.device), where
        # the arguments of a step that stay the same: the optimizer's own arrays and buffers
        names = ('exp_avg', 'exp_avg_sq', None, None) if self.state_bits == 32 else \
            ('exp_avg8', 'exp_rms8', 'exp_avg_scale', 'exp_rms_scale')
        self._fixed = tuple(ctypes.addressof(x) for x in (self._dtypes, self._sizes, self._where,
                                                          self._addresses)) + \
            (self._plan_host.data_ptr(), self._plan.data_ptr(), self.state_bits) + \
            tuple(None if n is None else self._state[n].data_ptr() for n in names) + \
            (self._state['master'].data_ptr() if 'master' in self._state else None,
             self._control.data_ptr())

    # -- hyper-parameters and state ----------------------------------------------------
    def set_lr(self, lr: float) -> None:
        """The learning rate of the steps queued behind this call (a store on the current stream; captured, a
        store of every replay)."""
        lr = float(lr)
        if not 0.0 <= lr < float('inf'):
            raise ValueError(f'the learning rate must be finite and not negative, got {lr}')
        # (behind a captured store, replays change the device's rate without the host)
        with torch.cuda.device(self.device):
            self._captured_lr |= torch.cuda.is_current_stream_capturing()
        if lr != self.lr or self._captured_lr:
            self.lr = lr
            self._lr.fill_(lr)

    @property
    def steps(self) -> int:
        """Steps taken (waits for the GPU: the counter is there, skipped steps do not count)."""
        return int(self._control[0].item())

    @property
    def state(self) -> Dict[str, torch.Tensor]:
        """The buffers by name (the optimizer's own: writing into them changes its state)."""
        return dict(self._state)

    def state_dict(self) -> Dict[str, object]:
        """Copies of the buffers, the step and, of 8-bit moments, the low 32 bits of the seed."""
        out = dict({k: v.clone() for k, v in self._state.items()}, step=self.steps)
        if self.state_bits == 8:
            out['seed'] = torch.tensor([self.seed & 0xffffffff])
        return out

    def load_state_dict(self, state: Dict[str, object]) -> None:
        """Copies the buffers of a `state_dict()` of the same parameters, `state_bits` and, if the state names one,
        `seed` (with another one the codes of the steps to come would be others)."""
        state = dict(state)
        seed = state.pop('seed', None) if self.state_bits == 8 else None
        if set(state) != set(self._state) | {'step'}:
            raise ValueError(f'the state has {sorted(state)}, expected {sorted(self._state)} and step')
        if seed is not None and int(seed) & 0xffffffff != self.seed & 0xffffffff:
            raise ValueError(f'the state is that of seed {int(seed)}, this optimizer has {self.seed}')
        for k, v in self._state.items():
            if tuple(state[k].shape) != tuple(v.shape) or state[k].dtype != v.dtype:
                raise ValueError(f'{k} must be {v.dtype} of {tuple(v.shape)}, got {state[k].dtype} '
                                 f'of {tuple(state[k].shape)}')
        self._write_control(int(state['step']))
        for k, v in self._state.items():
            v.view(torch.uint8).copy_(state[k].to(self.device).contiguous().view(torch.uint8))

    def zero_grad(self) -> None:
        """Drops the gradients (the next backward pass hands over fresh ones)."""
        for p in self.params:
            p.grad = None

    # -- one step ----------------------------------------------------------------------
    def step(self, grads: Optional[Sequence[Optional[torch.Tensor]]] = None,
             global_clip_norm: Optional[float] = None, guard: Optional[torch.Tensor] = None,
             guard_kind: int = 0, guard_host: Optional[torch.Tensor] = None
             ) -> Optional[torch.Tensor]:
        """Update every parameter from `grads` (default: their `.grad`).  With `global_clip_norm`
        the gradients are scaled to that norm if theirs is larger, and the norm before that is
        returned (one fp64 value on the device, overwritten by the next step).  `guard`, `guard_kind`,
        `guard_host`: as in `FlatOptimizer.step`; a skipped step changes nothing."""
        if self.device.index != torch._C._cuda_getDevice():
            with torch.cuda.device(self.device):
                return self.step(grads, global_clip_norm, guard, guard_kind, guard_host)
        if guard is not None and (guard.dtype != torch.float32 or guard.device != self.device
                                  or guard.numel() != 1):
            raise TypeError(f'the guard must be one float32 on {self.device}')
        if guard_host is not None and (guard_host.dtype != torch.float32 or guard_host.numel() != 1
                                       or guard_host.is_cuda):
            raise TypeError('guard_host must be one float32 in pinned host memory')
        clip = float(global_clip_norm or 0.0)
        if grads is not None and type(grads) is not list:
            grads = list(grads)
        step = hip.host().adamw_step
        while True:
            done = step(self.params, grads, *self._fixed, clip,
                        self.grad_norm.data_ptr() if clip else None, self.seed, hip.ptr(guard),
                        guard_kind if guard is not None else 0,
                        guard_host.data_ptr() if guard_host is not None else None,
                        self._workspace.data_ptr(), self._workspace.numel() * 8, hip.stream(),
                        self.device.index)
            if done:
                break
            if done is None:
                # captured: the plan is read by every replay
                if not any(p is self._plan for p in self._captured_plans):
                    self._captured_plans.append(self._plan)
                break
            # a parameter is not where it was
            if torch.cuda.is_current_stream_capturing():
                raise hip.HipLibraryError('a parameter has moved since the last step: take one '
                                          'eager step before capturing')
            self._make_plan()
        return self.grad_norm if clip else None

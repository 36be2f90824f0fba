"""AdamW over many tensors at once, its states in fp32 or in 8 bits (c1v_adamw_step of include/c1dvae.h).

    opt = AdamW(params, lr=1e-3, weight_decay=[0.01, 0.0, ...], clipnorm=10.0, states='8bit')
    loss.backward(); opt.step()              # or opt.step(grads)

One launch for the norm and one for the update, whatever the number of tensors (128 per launch).  The step number and the
learning rate live on the GPU, so a captured step can be replayed.  The reference's optimizers (Keras Nadam and RMSprop,
conv1d_text_vae.py:1328-1330) have neither decoupled weight decay nor 8-bit states.
"""
from __future__ import annotations

import ctypes as C
import math
import numbers
from array import array
from operator import attrgetter
from typing import Dict, List, Optional, Sequence, Union

import torch

from . import _lib as L

BLOCK = 128                     # state elements that share a scale
_CODE = {torch.float32: L.F32, torch.bfloat16: L.BF16}
_shape, _dtype = attrgetter('shape'), attrgetter('dtype')
_pointer, _device, _dense = torch.Tensor.data_ptr, torch.Tensor.get_device, torch.Tensor.is_contiguous
_KEYS = ('step', 'm', 'v', 'm_scale', 'v_scale')


class AdamW:
    """
    p' = (1 - lr wd) p - lr / (1 - b1^t) m' / (sqrt(v' / (1 - b2^t)) + eps) with m' = b1 m + (1 - b1) g, v' = b2 v + (1 - b2) g^2.

    params: contiguous float32 / bfloat16 tensors of one GPU that do not overlap; weight_decay: one number or one for each of
    them.  clipnorm > 0: all gradients together are scaled down to this norm where theirs is larger, and a step whose norm is
    not finite is left out (parameters, states and step number stay; `norm` holds it).

    states = '8bit': 2 bytes and 1/64 a weight instead of 8.  Blocks of 128 elements share a power-of-two scale; m is e4m3, v has
    five exponent and three mantissa bits, both are rounded stochastically from Philox(seed, step, element): the held
    moments follow the fp32 ones in the mean, and a run is reproducible bit by bit.  Within a block v reaches down to 2^-30 of
    its largest value; below that it is held as the smallest code, so that such a weight's steps are smaller than in fp32,
    never larger.
    """

    def __init__(self, params: Sequence[torch.Tensor], lr: float = 0.001, betas=(0.9, 0.999), eps: float = 1e-8,
                 weight_decay: Union[float, Sequence[float]] = 0.01, clipnorm: float = 0.0, states: str = 'f32', seed: int = 0):
        self.params: List[torch.Tensor] = list(params)
        if not self.params:
            raise ValueError('there are no parameters')
        decay = [float(weight_decay)] * len(self.params) if isinstance(weight_decay, numbers.Real) else [float(w) for w in weight_decay]
        if len(decay) != len(self.params):
            raise ValueError('weight_decay has {0} values for {1} parameters'.format(len(decay), len(self.params)))
        if states not in ('f32', '8bit'):
            raise ValueError("states must be 'f32' or '8bit', got {0!r}".format(states))
        b1, b2 = (float(b) for b in betas)
        whole = lambda x: 0 <= x < math.inf                       # (not NaN either)
        for name, value, fine in (('lr', lr, whole(lr)), ('betas', betas, 0 <= b1 < 1 and 0 <= b2 < 1), ('eps', eps, 1e-30 <= eps < math.inf),
                                  ('weight_decay', decay, all(whole(w) for w in decay)), ('clipnorm', clipnorm, whole(clipnorm))):
            if not fine:
                raise ValueError('the value of {0} is wrong: {1}'.format(name, value))
        for i, p in enumerate(self.params):
            self._check_param(i, p)
        self.device = self.params[0].device
        if self.device.type != 'cuda':
            raise L.C1VError('the parameters are on {0}: the HIP kernels are the only implementation of AdamW.'.format(self.device))
        spans = sorted((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size()) for p in self.params if p.numel())
        if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
            raise ValueError('parameters overlap in memory (the same tensor twice?)')
        self.betas, self.eps, self.clipnorm, self.seed = (b1, b2), float(eps), float(clipnorm), int(seed) % (1 << 64)
        self.states = states
        self._lib = L.load()
        n = len(self.params)
        table = (L.AdamwTensor * n)()
        at = chunk = 0
        for i, p in enumerate(self.params):
            table[i] = L.AdamwTensor(p.numel(), at, decay[i], chunk)
            at += -(-p.numel() // BLOCK) * BLOCK
            chunk += -(-p.numel() // L.ADAMW_CHUNK)
        if chunk >= 1 << 31:
            raise ValueError('too many weights')
        self._host = table
        self._table = torch.frombuffer(bytearray(bytes(table)), dtype=torch.uint8).to(self.device)
        self.weight_decay = decay
        at = max(at, BLOCK)
        e8 = states == '8bit'
        z = lambda k, dt: torch.zeros(k, dtype=dt, device=self.device)
        self.m = z(at, torch.float8_e4m3fn if e8 else torch.float32)
        self.v = z(at, torch.uint8 if e8 else torch.float32)
        self.m_scale = torch.full((at // BLOCK,), 1, dtype=torch.uint8, device=self.device) if e8 else None
        self.v_scale = torch.full((at // BLOCK,), 32, dtype=torch.uint8, device=self.device) if e8 else None
        self.t = z(1, torch.int64)
        self.norm = z(1, torch.float32).view(())
        self._lr = torch.tensor([float(lr)], dtype=torch.float64, device=self.device)
        self._sched = z(4, torch.float32)
        self._parts = L.ADAMW_PARTIALS * -(-n // L.ADAMW_GROUP)
        self._partial = z(self._parts if clipnorm > 0 else 1, torch.float64)
        self._shapes, self._kinds = [p.shape for p in self.params], [p.dtype for p in self.params]
        self._p_types = bytes(_CODE[k] for k in self._kinds)
        self._all_f32, self._no_bf16, self._where = [torch.float32] * n, bytes(n), [self.device.index] * n
        self._args = L.AdamwArgs(self._table.data_ptr(), C.addressof(table), n, 1 if e8 else 0, None, None,
                                 C.cast(self._p_types, C.c_void_p), None, self.m.data_ptr(),
                                 self.v.data_ptr(), self.m_scale.data_ptr() if e8 else None, self.v_scale.data_ptr() if e8 else None,
                                 self.t.data_ptr(), self._lr.data_ptr(), b1, b2, self.eps, self.clipnorm, 1.0, self._sched.data_ptr(),
                                 self._partial.data_ptr(), self._parts, self.norm.data_ptr(), None, self.seed)

    def _check_param(self, i: int, p: torch.Tensor):
        if p.dtype not in _CODE:
            raise ValueError('parameter {0} must be float32 or bfloat16, got {1}'.format(i, p.dtype))
        if not p.is_contiguous():
            raise ValueError('parameter {0} is not contiguous'.format(i))
        if p.device != self.params[0].device:
            raise ValueError('parameter {0} is on {1}, parameter 0 on {2}'.format(i, p.device, self.params[0].device))

    # ---- learning rate, state ------------------------------------------------------------------------------
    def set_lr(self, lr: float):
        if not 0 <= lr < math.inf:
            raise ValueError('the value of lr is wrong: {0}'.format(lr))
        self._lr.fill_(float(lr))

    def get_lr(self) -> float:
        return float(self._lr.item())

    def reset(self):
        """Back to step 0 with empty states."""
        for x in (self.m, self.v, self.t):
            x.view(torch.uint8).zero_()

    def state_tensors(self) -> List[torch.Tensor]:
        """What a step changes beside the parameters (to be saved around a warm-up run)."""
        return [x for x in (self.t, self._lr, self.m, self.v, self.m_scale, self.v_scale) if x is not None]

    def state_dict(self) -> Dict[str, Optional[torch.Tensor]]:
        return {k: None if x is None else x.clone() for k, x in zip(_KEYS, (self.t, self.m, self.v, self.m_scale, self.v_scale))}

    def load_state_dict(self, state: Dict[str, Optional[torch.Tensor]]):
        own = dict(zip(_KEYS, (self.t, self.m, self.v, self.m_scale, self.v_scale)))
        for k, x in own.items():
            s = state[k]
            if (s is None) != (x is None) or (x is not None and (s.dtype != x.dtype or s.numel() != x.numel())):
                raise ValueError('state `{0}` does not belong to this optimizer'.format(k))
        for k, x in own.items():
            if x is not None:
                x.copy_(state[k].reshape(x.shape))

    def moments(self, i: int):
        """(m, v) of parameter i in float32, in its shape."""
        d, shape = self._host[i], self.params[i].shape
        a, b = d.offset, d.offset + -(-d.n // BLOCK) * BLOCK
        m, v = self.m[a:b], self.v[a:b]
        if self.states == '8bit':
            ms, vs = (s[a // BLOCK:b // BLOCK].to(torch.int32).unsqueeze(1) for s in (self.m_scale, self.v_scale))
            m = (m.float().view(-1, BLOCK) * (ms << 23).view(torch.float32)).view(-1)
            c = v.to(torch.int32).view(-1, BLOCK)
            x = ((c + 8 * vs - 240) << 20).view(torch.float32)
            v = torch.where(c == 0, 0.0, torch.where(c == 255, float('nan'), x)).view(-1)
        return m[:d.n].view(shape).clone(), v[:d.n].view(shape).clone()

    # ---- step ------------------------------------------------------------------------------------------------
    def args(self, grads: Sequence[Optional[torch.Tensor]], grad_scale: float = 1.0, ctr: Optional[int] = None) -> 'L.AdamwArgs':
        """The argument struct of c1v_adamw_step for these gradients (for a recorded step: valid while they and this optimizer
        live, and until the next call of `args` or `step`)."""
        params, grads = self.params, list(grads)
        # (whole lists at a time: a loop over tensors costs more than the launches.  `.data` may have been replaced since.)
        if list(map(_shape, params)) != self._shapes or list(map(_dtype, params)) != self._kinds or \
                list(map(_device, params)) != self._where or not all(map(_dense, params)):
            raise ValueError('the parameters changed their number, or one its type, shape, layout or device')
        if len(grads) != len(params):
            raise ValueError('{0} gradients for {1} parameters'.format(len(grads), len(params)))
        if type(None) not in map(type, grads) and list(map(_shape, grads)) == self._shapes and list(map(_dtype, grads)) == self._all_f32 and \
                list(map(_device, grads)) == self._where and all(map(_dense, grads)):
            G, GT = map(_pointer, grads), self._no_bf16
        else:
            G, GT = self._mixed_grads(grads)
        self._alive = grads
        self._pointers = P, G, GT = array('Q', map(_pointer, params)), array('Q', G), array('B', GT)
        if not math.isfinite(grad_scale):
            raise ValueError('the value of grad_scale is wrong: {0}'.format(grad_scale))
        a = self._args
        a.p, a.g = P.buffer_info()[0], G.buffer_info()[0]
        a.g_dtype = GT.buffer_info()[0]
        a.grad_scale, a.ctr = grad_scale, ctr
        return a

    def _mixed_grads(self, grads: list):
        """Pointers and types of gradients of which some are missing, bfloat16 or strided (replaced by a copy in `grads`)."""
        G, GT = [], []
        for i, (g, shape, where) in enumerate(zip(grads, self._shapes, self._where)):
            if g is None:
                G.append(0)
                GT.append(0)
                continue
            if g.shape != shape or g.dtype not in _CODE or g.get_device() != where:
                raise ValueError('gradient {0} is {1} {2} on {3}, its parameter {4} on {5}'.format(i, tuple(g.shape), g.dtype, g.device, tuple(shape), self.device))
            if not g.is_contiguous():
                grads[i] = g = g.detach().contiguous()
            G.append(g.data_ptr())
            GT.append(_CODE[g.dtype])
        return G, GT

    def step(self, grads: Optional[Sequence[Optional[torch.Tensor]]] = None, grad_scale: float = 1.0):
        """One step on the current stream.  grads: one tensor (float32 or bfloat16) for each parameter, or None to leave that
        parameter out; without the argument, the parameters' `.grad`.  grad_scale multiplies every gradient (1 / ranks after a
        sum over them)."""
        a = self.args([p.grad for p in self.params] if grads is None else grads, grad_scale)
        i = self.device.index
        if torch._C._cuda_getDevice() == i:
            rc = self._lib.c1v_adamw_step(C.byref(a), torch._C._cuda_getCurrentRawStream(i))
        else:
            with torch.cuda.device(i):
                rc = self._lib.c1v_adamw_step(C.byref(a), torch._C._cuda_getCurrentRawStream(i))
        self._alive = None                                       # (copies of strided gradients are freed in stream order)
        if rc:
            L.check(rc, 'c1v_adamw_step')
        torch.autograd.graph.increment_version(self.params)      # as any change in place

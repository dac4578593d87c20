"""The AdamW step of a training run on the MI355X, over all parameters at once
(``hi2x_adamw_step``), with the moments in 32 bits or in 8.

It updates what :mod:`hi2_amd.qad_kernel` trains (latents and ladder bytes, ``hi2/qad.py``) and the
weights of :mod:`hi2_amd.experts`: one launch for up to 192 tensors, whatever their sizes, the
host never waiting."""

from __future__ import annotations

import numpy as np
import torch

from . import _lib

__all__ = ["AdamW"]

BLOCK = 256  # HI2X_ADAMW_BLOCK: elements that share a unit of 8-bit moments
CHUNK = 4096  # HI2X_ADAMW_CHUNK
DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}

_TENSOR = np.dtype([("n", "<i8"), ("start", "<i8"), ("first_chunk", "<i8"), ("group", "<i4"),
                    ("reserved", "<i4")])


def _tensors():
    """The host extension; raises where it is not built."""
    try:
        from . import _tensors as module
    except ImportError as e:
        raise RuntimeError(f"hi2_amd/_tensors.so is not built or does not load ({e}): run "
                           "`python -m hi2_amd.build`") from e
    return module


class _Set:
    """The parameters of one type: their table on the host and on the device."""

    def __init__(self, dtype, entries, dev):
        self.dtype = dtype
        self.params = [p for p, _, _ in entries]
        self.sizes = np.array([p.numel() for p in self.params], dtype=np.int64)
        self.addresses = np.zeros((2, len(entries)), dtype=np.uint64)  # written in every step
        table = np.zeros(len(entries), dtype=_TENSOR)
        chunk = 0
        for i, (p, start, group) in enumerate(entries):
            table[i] = (p.numel(), start, chunk, group, 0)
            chunk += -(-p.numel() // CHUNK)
        self.table = table
        self.device_table = _lib.h2d(torch.from_numpy(table.view(np.uint8).copy()), dev)


class AdamW(torch.optim.Optimizer):
    """AdamW over contiguous float32, float16 or bfloat16 parameters of one device::

        m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2
        p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)

    in float32 with one rounding to the parameter's type.  Options may differ between parameter
    groups and change between steps; ``lr`` is a number or a float32 tensor of one element on the
    device (a captured step reads the tensor anew in every replay, and keeps numbers as they were).
    A parameter without a gradient is left as it is, its count of steps too; the counts are on
    the device, so a captured step counts on in its replays.

    * ``state_bits=8``: moments take two bytes a parameter in the place of eight.  256 neighbours
      share a unit; a moment is +-q^2 units and the root of a second moment q^2 units (q up to 127
      and 255), rounded to the nearest q, a root that is not zero to no less than 1.  The step
      itself uses the new moments before that rounding.  A block whose largest moment is not finite
      becomes NaN.
    * ``master=True``: float16 and bfloat16 parameters keep a float32 copy that takes the steps and
      is rounded to them (without it, steps below half their spacing are lost).  It is made from
      the parameters at construction and by :meth:`load_masters`.

    Moments (and masters) of all parameters lie in one buffer each, in the order of the groups,
    every parameter from a multiple of 256 elements on (:attr:`starts`).  Parameters cannot be
    added, and their types and sizes not changed, after construction.  Options of other AdamW
    variants (``amsgrad``, ``maximize``, ``differentiable``, ``decoupled_weight_decay=False``) are
    refused in a group or a state; what else a group holds (names, what a scheduler keeps there)
    stays there."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, state_bits: int = 32, master: bool = False):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits {state_bits} (8 or 32)")
        self._laid_out = False
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))
        self.state_bits = state_bits
        every = [(p, gi) for gi, g in enumerate(self.param_groups) for p in g["params"]]
        dev = _lib.require_gpu(*(p for p, _ in every))
        self.device = dev
        starts, at = [], 0
        by_type: dict = {}
        for p, gi in every:
            if p.dtype not in DTYPES:
                raise ValueError(f"a parameter is {p.dtype} (float32, float16 or bfloat16)")
            if not p.is_contiguous():
                raise ValueError(f"a parameter of shape {tuple(p.shape)} is not contiguous")
            starts.append(at)
            if p.numel():
                by_type.setdefault(p.dtype, []).append((p, at, gi))
            at += -(-p.numel() // BLOCK) * BLOCK
        spans = sorted((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size())
                       for p, _ in every if p.numel())
        if any(b < end for (_, end), (b, _) in zip(spans, spans[1:])):
            raise ValueError("two parameters share memory, or one is there twice")
        #: the first element of each parameter in the buffers
        self.starts = starts
        self._params = [p for p, _ in every]
        self._blocks = at // BLOCK
        kind = torch.float32 if state_bits == 32 else torch.uint8
        self._m = torch.zeros(at, dtype=kind, device=dev)
        self._v = torch.zeros(at, dtype=kind, device=dev)
        self._units = torch.zeros(2, self._blocks, dtype=torch.float32, device=dev) \
            if state_bits == 8 else None
        self._sets = [_Set(d, entries, dev) for d, entries in by_type.items()]
        self._types = [str(p.dtype) for p in self._params]
        self._numels = [p.numel() for p in self._params]
        count = sum(len(s.params) for s in self._sets)
        self._steps = torch.zeros(count, dtype=torch.int64, device=dev)
        self._done = torch.zeros(count, dtype=torch.int32, device=dev)
        #: float32 parameters in the buffers' layout, or None
        self.master = None
        if master and any(s.dtype != torch.float32 for s in self._sets):
            self.master = torch.zeros(at, dtype=torch.float32, device=dev)
            self.load_masters()
        self._laid_out = True
        for g in self.param_groups:
            self._options(g)

    @staticmethod
    def _counted(types, numels) -> list:
        """The parameters in the order of their counts of steps: type after type, the empty ones
        left out."""
        live = [i for i, n in enumerate(numels) if n]
        return [i for t in dict.fromkeys(types[i] for i in live) for i in live if types[i] == t]

    def add_param_group(self, param_group):
        if self._laid_out:
            raise RuntimeError("AdamW: parameters cannot be added after construction")
        super().add_param_group(param_group)

    def __getstate__(self):
        raise TypeError("AdamW is not copied or pickled, which would leave its moments behind: take "
                        "its state_dict")

    def _options(self, g) -> tuple:
        """A group's options as ``hi2x_adamw_group``, checked."""
        lr, (b1, b2), eps, wd = g["lr"], g["betas"], g["eps"], g["weight_decay"]
        for name, given in (("amsgrad", False), ("maximize", False), ("differentiable", False),
                            ("decoupled_weight_decay", True)):
            if bool(g.get(name, given)) is not given:
                raise ValueError(f"AdamW has no {name}={g[name]}")
        tensor = None
        if isinstance(lr, torch.Tensor):
            if lr.device != self.device or lr.dtype != torch.float32 or lr.numel() != 1:
                raise ValueError(f"lr is a {lr.dtype} tensor of {lr.numel()} elements on "
                                 f"{lr.device}: one float32 on {self.device} expected")
            tensor, lr = lr.data_ptr(), 0.0
        if not lr >= 0 or not eps >= 0 or not wd >= 0 or not 0 <= b1 < 1 or not 0 <= b2 < 1:
            raise ValueError(f"lr {lr}, betas {(b1, b2)}, eps {eps}, weight_decay {wd}: lr, eps "
                             "and weight_decay not below 0 and betas in [0, 1) expected")
        return lr, b1, b2, eps, wd, tensor

    @torch.no_grad()
    def step(self, closure=None):
        """One step with the gradients in ``p.grad``, enqueued on the current stream.  To autograd it
        is a write in place: a backward that still needs the old parameters raises."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        groups = (_lib.AdamwGroup * len(self.param_groups))(
            *(_lib.AdamwGroup(*self._options(g)) for g in self.param_groups))
        odd = []  # gradients made contiguous, alive until they are read
        for s in self._sets:  # (all of them before the first launch: a step is taken whole or not)
            at_p, at_g = s.addresses[0].ctypes.data, s.addresses[1].ctypes.data
            for i in _tensors().addresses(s.params, s.sizes.ctypes.data, DTYPES[s.dtype],
                                          self.device.index, at_p, at_g):
                odd.append(s.params[i].grad.contiguous())
                s.addresses[1, i] = odd[-1].data_ptr()
        at = 0
        units = self._units
        for s in self._sets:
            n = len(s.params)
            _lib.call("hi2x_adamw_step", self.device, s.table.ctypes.data,
                      s.device_table.data_ptr(), s.addresses[0].ctypes.data,
                      s.addresses[1].ctypes.data, n, DTYPES[s.dtype], self.state_bits, groups,
                      len(groups), self._m.data_ptr(), self._v.data_ptr(),
                      None if units is None else units[0].data_ptr(),
                      None if units is None else units[1].data_ptr(),
                      None if self.master is None or s.dtype == torch.float32
                      else self.master.data_ptr(),
                      self._steps[at:].data_ptr(), self._done[at:].data_ptr())
            _tensors().stepped(s.params, s.addresses[1].ctypes.data)
            at += n
        return loss

    def moments(self) -> tuple[torch.Tensor, torch.Tensor]:
        """The first and second moments of all parameters, float32 in the buffers' layout: with
        32 bits the buffers themselves, with 8 the values they stand for."""
        if self.state_bits == 32:
            return self._m, self._v
        m = torch.empty(2, self._m.numel(), dtype=torch.float32, device=self.device)
        _lib.call("hi2x_adamw_moments", self.device, self._m.data_ptr(), self._v.data_ptr(),
                  self._units[0].data_ptr(), self._units[1].data_ptr(), self._blocks,
                  m[0].data_ptr(), m[1].data_ptr())
        return m[0], m[1]

    @torch.no_grad()
    def load_moments(self, m: torch.Tensor, v: torch.Tensor, step: int | None = None) -> None:
        """Take over float32 moments in the buffers' layout (what :meth:`moments` gives, of
        either width), and a count of steps for every parameter.  What lies between a parameter's
        end and the next multiple of 256 is taken as zero."""
        for name, t in (("m", m), ("v", v)):
            if t.shape != self._m.shape or t.dtype != torch.float32 or t.device != self.device:
                raise ValueError(f"{name} is {t.dtype} {tuple(t.shape)} on {t.device}, expected "
                                 f"float32 {tuple(self._m.shape)} on {self.device}")
        if step is not None and step < 0:
            raise ValueError(f"step {step}")
        gaps = self._gaps()
        m, v = m.clone().index_fill_(0, gaps, 0.0), v.clone().index_fill_(0, gaps, 0.0)
        if self.state_bits == 32:
            self._m.copy_(m)
            self._v.copy_(v)
        else:
            _lib.call("hi2x_adamw_hold", self.device, m.data_ptr(), v.data_ptr(), self._blocks,
                      self._m.data_ptr(), self._v.data_ptr(), self._units[0].data_ptr(),
                      self._units[1].data_ptr())
        if step is not None:
            self._steps.fill_(step)

    def _gaps(self) -> torch.Tensor:
        """The elements of the buffers that belong to no parameter."""
        gaps = [np.arange(a + p.numel(), a + -(-p.numel() // BLOCK) * BLOCK)
                for a, p in zip(self.starts, self._params)]
        return _lib.h2d(torch.from_numpy(np.concatenate(gaps or [np.zeros(0, np.int64)])
                                         .astype(np.int64)), self.device)

    @torch.no_grad()
    def load_masters(self) -> None:
        """Make the masters anew from the parameters (after these were loaded from elsewhere)."""
        if self.master is None:
            raise RuntimeError("AdamW: there are no masters")
        for a, p in zip(self.starts, self._params):
            self.master[a:a + p.numel()].copy_(p.detach().reshape(-1))

    def state_dict(self) -> dict:
        """The options and the state: the buffers themselves, not copies of them."""
        out = super().state_dict()
        out["state"] = dict(state_bits=self.state_bits, starts=list(self.starts),
                            sizes=list(self._numels), types=list(self._types), m=self._m,
                            v=self._v, units=self._units, steps=self._steps, master=self.master)
        return out

    @torch.no_grad()
    def load_state_dict(self, state_dict: dict) -> None:
        """Take over a :meth:`state_dict` of an optimizer over the same parameters and of the same
        ``state_bits`` and ``master``; the parameters' types may be others.  A learning rate that is
        a tensor here stays that tensor and takes the value."""
        given = state_dict["state"]
        mine = self.state_dict()["state"]
        if given["state_bits"] != self.state_bits or list(given["starts"]) != self.starts or \
                list(given.get("sizes", self._numels)) != self._numels:
            raise ValueError("load_state_dict: the state is of other parameters or another width")
        if [(len(g["params"])) for g in state_dict["param_groups"]] != \
                [len(g["params"]) for g in self.param_groups]:
            raise ValueError("load_state_dict: other parameter groups")
        for name in ("m", "v", "units", "steps", "master"):
            a, b = mine[name], given[name]
            if (a is None) != (b is None) or a is not None and (a.shape != b.shape or
                                                                a.dtype != b.dtype):
                raise ValueError(f"load_state_dict: {name} does not fit")
        steps = given["steps"]
        theirs = self._counted(given.get("types", self._types), self._numels)
        ours = self._counted(self._types, self._numels)
        if theirs != ours:  # counts lie type after type
            at = {p: i for i, p in enumerate(theirs)}
            steps = steps[torch.tensor([at[p] for p in ours], device=steps.device)]
        taken = []
        for g, h in zip(self.param_groups, state_dict["param_groups"]):
            options = {k: v for k, v in h.items() if k != "params"}
            if isinstance(options.get("lr"), torch.Tensor):
                options["lr"] = options["lr"].to(self.device, copy=True)
            self._options({**g, **options})
            taken.append(options)
        for g, options in zip(self.param_groups, taken):
            if isinstance(g["lr"], torch.Tensor) and "lr" in options:
                lr = options.pop("lr")  # (the tensor stays: captured steps read it)
                g["lr"].copy_(lr) if isinstance(lr, torch.Tensor) else g["lr"].fill_(lr)
            g.update(options)
        self._steps.copy_(steps)
        for name in ("m", "v", "units", "master"):
            if mine[name] is not None:
                mine[name].copy_(given[name])

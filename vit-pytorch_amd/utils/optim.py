"""Optimizer step of the fine-tuning loop on the HIP kernel library.

The reference loop (train.py:535-538) runs, per optimisation step,

    torch.nn.utils.clip_grad_norm_(model.parameters(), args.max_grad_norm)
    optimizer.step()            # torch.optim.SGD(lr, momentum=0.9, weight_decay) built at train.py:475-478
    scheduler.step()
    optimizer.zero_grad()

`FusedSGD` is a `torch.optim.Optimizer` (so the LambdaLR schedules of utils/scheduler.py drive it
unchanged) whose `step(max_grad_norm=...)` does the clipping and the update in two kernel launches
over a table of all tensors (`vitk_sgd_norm_sq`, `vitk_sgd_step`).  Same arithmetic as
torch.optim.SGD without Nesterov: the momentum buffer starts as the first (clipped) gradient.
There is no CPU path: the tensors must live on the GPU and the kernel library must load.
"""
import ctypes
from operator import attrgetter

import numpy as np
import torch

import vitk

_ENTRY = np.dtype([("param", "<u8"), ("grad", "<u8"), ("mom", "<u8"), ("n", "<i8"), ("block0", "<i4"), ("flags", "<i4")])
_CHUNK = 8192            # elements per block (kernel constant)
assert _ENTRY.itemsize == 40


class FusedSGD(torch.optim.Optimizer):
    def __init__(self, params, lr, momentum=0.0, dampening=0.0, weight_decay=0.0):
        if lr < 0.0 or momentum < 0.0 or weight_decay < 0.0:
            raise ValueError("lr, momentum and weight_decay must be non-negative")
        super().__init__(params, dict(lr=lr, momentum=momentum, dampening=dampening, weight_decay=weight_decay))
        self._slots = None
        self._dev = None          # the table on the device
        self._last = None         # its contents (numpy), to skip uploads of an unchanged table
        self._ring, self._turn = [], 0

    def _table(self, group):
        rows = []
        block0 = 0
        for p in group["params"]:
            g = p.grad
            if g is None:
                continue
            if not (p.is_cuda and p.dtype == torch.float32 and g.dtype == torch.float32
                    and p.is_contiguous() and g.is_contiguous()):
                raise ValueError("FusedSGD needs contiguous fp32 parameters and gradients on the GPU")
            st = self.state[p]
            first = 0
            if group["momentum"] != 0.0:
                if "momentum_buffer" not in st:
                    st["momentum_buffer"] = torch.empty_like(p, memory_format=torch.contiguous_format)
                    first = 1
                m = st["momentum_buffer"].data_ptr()
            else:
                m = 0
            n = p.numel()
            vec = 2 if (n % 4 == 0 and (p.data_ptr() | g.data_ptr() | m) % 16 == 0) else 0
            rows.append((p.data_ptr(), g.data_ptr(), m, n, block0, first | vec))
            block0 += (n + _CHUNK - 1) // _CHUNK
        return rows, block0

    @torch.no_grad()
    def step(self, closure=None, max_grad_norm=None):
        """One update.  With `max_grad_norm`, gradients of ALL groups are clipped by their joint
        2-norm first (clip_grad_norm_ semantics) and that norm is returned as a 0-d tensor."""
        if closure is not None:
            raise ValueError("FusedSGD does not re-evaluate the model")
        tables = [self._table(g) for g in self.param_groups]
        n_rows = sum(len(r) for r, _ in tables)
        if n_rows == 0:
            return None
        dev = next(p for g in self.param_groups for p in g["params"] if p.grad is not None).device
        multi = len([1 for r, _ in tables if r]) > 1
        need = n_rows * (2 if multi else 1)
        # rows [0, n_rows): every group, blocks numbered globally (norm pass; also the update of a
        # single group).  With several groups, rows [n_rows, 2 n_rows) repeat them numbered per group.
        host = np.zeros(need, dtype=_ENTRY)
        at, blk = 0, 0
        spans = []
        for rows, nblk in tables:
            for r in rows:
                host[at] = r[:4] + (r[4] + blk, r[5])
                if multi:
                    host[n_rows + at] = r
                at += 1
            spans.append(((n_rows if multi else 0) + at - len(rows), len(rows), nblk))
            blk += nblk
        # The caching allocator hands the same gradient addresses back step after step, so the table
        # on the device is usually still right: upload only when it changed.  Uploads go through a
        # ring of pinned buffers, each guarded by an event, so the host never waits for the GPU to
        # catch up with the step it has just enqueued.
        if self._last is None or self._last.shape != host.shape or not np.array_equal(self._last, host):
            nbytes = need * _ENTRY.itemsize
            if self._dev is None or self._dev.numel() < nbytes:
                self._dev = torch.empty(nbytes, dtype=torch.uint8, device=dev)
                self._ring = []
            if not self._ring or self._ring[0][0].numel() < nbytes:
                # pinning memory synchronises the device: take all four buffers at once, with head room
                self._ring = [(torch.empty(max(2 * nbytes, 1 << 14), dtype=torch.uint8).pin_memory(), torch.cuda.Event())
                              for _ in range(4)]
                self._turn = 0
            else:
                self._ring[self._turn][1].synchronize()      # that upload was enqueued four changes ago
            buf, ev = self._ring[self._turn]
            buf.numpy()[:nbytes] = host.view(np.uint8)
            self._dev[:nbytes].copy_(buf[:nbytes], non_blocking=True)
            ev.record()
            self._turn = (self._turn + 1) % 4
            self._last = host
        if self._slots is None:
            self._slots = torch.zeros(64 + 1024, dtype=torch.float32, device=dev)      # VITK_SGD_SLOTS (include/vitk.h)
        stream = ctypes.c_void_p(torch.cuda.current_stream(dev).cuda_stream)
        base = self._dev.data_ptr()
        slots = None
        if max_grad_norm is not None:
            vitk.check(vitk.lib.vitk_sgd_norm_sq(base, n_rows, blk, self._slots.data_ptr(), stream), "sgd_norm_sq")
            slots = self._slots.data_ptr()
        for (first_row, cnt, nblk), group in zip(spans, self.param_groups):
            if cnt == 0:
                continue
            vitk.check(vitk.lib.vitk_sgd_step(base + first_row * _ENTRY.itemsize, cnt, nblk, slots,
                                              float(max_grad_norm or 0.0), float(group["lr"]),
                                              float(group["momentum"]), float(group["dampening"]),
                                              float(group["weight_decay"]), stream), "sgd_step")
        # the parameters were written through raw pointers: renew the GEMM operands kept with them (one launch)
        vitk.ops.refresh_operands([p for g in self.param_groups for p in g["params"] if p.grad is not None])
        if max_grad_norm is not None:
            return self._slots[0].sqrt()
        return None


_ADAMW_ENTRY = np.dtype([("param", "<u8"), ("grad", "<u8"), ("m", "<u8"), ("v", "<u8"), ("m_scale", "<u8"),
                         ("v_scale", "<u8"), ("n", "<i8"), ("block0", "<i4"), ("flags", "<i4")])
_ADAMW_SLOTS = 1 + 8192      # VITK_ADAMW_SLOTS (include/vitk.h)
_SCALE_BLOCK = 256           # elements of an 8-bit state that share a scale
assert _ADAMW_ENTRY.itemsize == 64


class FusedAdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay) over all tensors in one launch, with gradient clipping by the joint norm.

    ``state_bits`` 32: moments in fp32, the arithmetic and the state names of torch.optim.AdamW (`exp_avg`, `exp_avg_sq`),
    whose state dicts it loads.  8: e4m3 codes of the parameter's shape with one fp32 scale for each 256 consecutive
    elements (`exp_avg_scale`, `exp_avg_sq_scale`); an element of `exp_avg` is code * scale, of `exp_avg_sq`
    (code * scale)^2.  Codes are rounded at random from (``seed``, step, element), so that their expectation is the
    moment (but for roots below 2^-9 of a scale, which are held as 2^-9); a moment that is no finite number is held as NaN, alone.
    Replicas with equal gradients stay bit-identical.  Parameters and gradients are contiguous fp32 tensors on
    one GPU.  A step counts on the host, so it is not captured into a graph."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, seed=0):
        if lr < 0.0 or eps < 0.0 or weight_decay < 0.0:
            raise ValueError("lr, eps and weight_decay must be non-negative")
        if not all(0.0 <= b < 1.0 for b in betas):
            raise ValueError("betas lie in [0, 1)")
        if state_bits not in (8, 32):
            raise ValueError("state_bits is 8 or 32")
        self.state_bits, self.seed = state_bits, int(seed) & 0xFFFFFFFF
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay))
        self._empty()

    def _empty(self):
        self._slots = None
        self._dev = None          # the table on the device
        self._last = None         # its contents (numpy), to skip uploads of an unchanged table
        self._ring, self._turn = [], 0

    def __getstate__(self):       # copies and pickles: the settings, and buffers of their own
        return dict(super().__getstate__(), state_bits=self.state_bits, seed=self.seed)

    def __setstate__(self, state):
        super().__setstate__(state)
        if "_ring" not in self.__dict__:                 # (not when load_state_dict() comes this way)
            self._empty()

    def load_state_dict(self, state_dict):
        held = [s for s in state_dict["state"].values() if s]
        if any(("exp_avg_scale" in s) != (self.state_bits == 8) for s in held):
            raise ValueError(f"the state dict's moments are not in {self.state_bits} bits")
        if any(g.get("amsgrad") or g.get("maximize") for g in state_dict["param_groups"]):
            raise ValueError("FusedAdamW has no amsgrad and no maximize")
        # (super() pairs groups and parameters in this order, and refuses others)
        ours = [p for g in self.param_groups for p in g["params"]]
        for key, p in zip([k for g in state_dict["param_groups"] for k in g["params"]], ours):
            st = state_dict["state"].get(key)
            if st and not self._fits(p, st):
                raise ValueError(f"the state dict's moments do not belong to a parameter of shape {tuple(p.shape)}")
        super().load_state_dict(state_dict)
        for p, st in self.state.items():
            if st:
                st["step"] = int(st["step"])
                kind = torch.float8_e4m3fn if self.state_bits == 8 else torch.float32      # exact: codes came back as fp32
                for name, value in st.items():
                    if name != "step":      # copies: the state dict's tensors may be another optimizer's
                        st[name] = torch.empty(value.shape, dtype=torch.float32 if name.endswith("_scale") else kind,
                                               device=p.device).copy_(value)

    def _fits(self, p, st):
        """Whether these states have the sizes that the kernel takes for granted."""
        if not all(name in st and st[name].shape == p.shape for name in ("exp_avg", "exp_avg_sq")):
            return False
        return self.state_bits != 8 or all(name in st and st[name].numel() == -(-p.numel() // _SCALE_BLOCK)
                                           for name in ("exp_avg_scale", "exp_avg_sq_scale"))

    def _begin(self, p, st):
        """Empty states of a parameter: the first step takes them as zeros."""
        kind = torch.float8_e4m3fn if self.state_bits == 8 else torch.float32
        st["step"] = 0
        st["exp_avg"] = torch.empty(p.shape, dtype=kind, device=p.device)
        st["exp_avg_sq"] = torch.empty(p.shape, dtype=kind, device=p.device)
        if self.state_bits == 8:
            for name in ("exp_avg_scale", "exp_avg_sq_scale"):
                st[name] = torch.empty(-(-p.numel() // _SCALE_BLOCK), dtype=torch.float32, device=p.device)

    def _table(self, ps, grads, sts, sizes):
        """The rows of all tensors, column by column, with blocks counted from 0; (table, number of blocks)."""
        host = np.zeros(len(ps), dtype=_ADAMW_ENTRY)
        host["param"] = [p.data_ptr() for p in ps]
        host["grad"] = [g.data_ptr() for g in grads]
        host["m"] = [s["exp_avg"].data_ptr() for s in sts]
        host["v"] = [s["exp_avg_sq"].data_ptr() for s in sts]
        if self.state_bits == 8:
            host["m_scale"] = [s["exp_avg_scale"].data_ptr() for s in sts]
            host["v_scale"] = [s["exp_avg_sq_scale"].data_ptr() for s in sts]
        host["n"] = sizes
        blocks = np.cumsum((host["n"] + (_CHUNK - 1)) // _CHUNK)
        host["block0"][1:] = blocks[:-1]
        vec = ((host["param"] | host["grad"]) % 16 == 0) & ((host["m"] | host["v"]) % (4 if self.state_bits == 8 else 16) == 0)
        host["flags"] = vec * 2
        host["flags"] |= np.array([s["step"] == 0 for s in sts])
        return host, blocks

    def _upload(self, host, blocks, dev):
        """The table and, behind it, the entry of each block, on the device; uploads go through a ring of pinned buffers,
        each guarded by an event, so the host never waits for the step it has just enqueued."""
        if self._dev is not None and self._dev.device != dev:          # the model has moved
            self._dev = self._last = self._slots = None
            self._ring = []
        if self._last is not None and self._last.shape == host.shape and np.array_equal(self._last, host):
            return
        entry_of = np.repeat(np.arange(len(host), dtype=np.int32), np.diff(blocks, prepend=0))
        nbytes = host.nbytes + entry_of.nbytes
        if self._dev is None or self._dev.numel() < nbytes:
            self._dev = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        if not self._ring or self._ring[0][0].numel() < nbytes:
            self._ring = [(torch.empty(max(2 * nbytes, 1 << 14), dtype=torch.uint8, pin_memory=True), torch.cuda.Event())
                          for _ in range(4)]
            self._turn = 0
        else:
            self._ring[self._turn][1].synchronize()
        buf, ev = self._ring[self._turn]
        buf.numpy()[:host.nbytes] = host.view(np.uint8)
        buf.numpy()[host.nbytes:nbytes] = entry_of.view(np.uint8)
        self._dev[:nbytes].copy_(buf[:nbytes], non_blocking=True)
        ev.record()
        self._turn = (self._turn + 1) % 4
        self._last = host

    @torch.no_grad()
    def step(self, closure=None, max_grad_norm=None):
        """One update.  With `max_grad_norm`, gradients of ALL groups are clipped by their joint 2-norm first and that
        norm is returned as a 0-d tensor."""
        if closure is not None:
            raise ValueError("FusedAdamW does not re-evaluate the model")
        if max_grad_norm is not None and not max_grad_norm >= 0.0:
            raise ValueError("max_grad_norm must be non-negative")
        # (loops over bound methods of the class: with a few hundred small tensors this function is what a step costs)
        state, Tensor = self.state, torch.Tensor
        groups = []
        for group in self.param_groups:
            pairs = [(p, g) for p in group["params"] if (g := p.grad) is not None and g.numel()]
            groups.append(([p for p, _ in pairs], [g for _, g in pairs]))
        all_ps, all_grads = sum((ps for ps, _ in groups), []), sum((grads for _, grads in groups), [])
        if not all_ps:
            return None
        dev, both = all_ps[0].device, all_ps + all_grads
        if (dev.type != "cuda" or any(map(attrgetter("is_sparse"), all_grads)) or set(map(attrgetter("dtype"), both)) != {torch.float32}
                or set(map(Tensor.get_device, both)) != {dev.index} or not all(map(Tensor.is_contiguous, both))):
            raise ValueError("FusedAdamW needs contiguous fp32 parameters and gradients on one GPU")
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("FusedAdamW.step counts steps on the host and is not captured into a graph")
        # one launch for the tensors of a group that have taken the same number of steps
        all_ps, all_grads, all_sts, spans = [], [], [], []
        for group, (ps, grads) in zip(self.param_groups, groups):
            sts = [state[p] for p in ps]
            for p, st in zip(ps, sts):
                if not st:
                    self._begin(p, st)
            steps = [st["step"] for st in sts]
            for t in dict.fromkeys(steps):
                of_t = (ps, grads, sts)
                if steps.count(t) != len(steps):
                    of_t = ([x for x, n in zip(xs, steps) if n == t] for xs in of_t)
                at = len(all_ps)
                for xs, more in zip((all_ps, all_grads, all_sts), of_t):
                    xs += more
                spans.append((group, t, at, len(all_ps) - at))
        # a parameter may have got another tensor, or moved, since its gradient or its states were made
        moments = [st["exp_avg"] for st in all_sts]
        sizes = list(map(Tensor.numel, all_ps))
        if (sizes != list(map(Tensor.numel, moments)) or sizes != list(map(Tensor.numel, all_grads))
                or set(map(Tensor.get_device, moments)) != {dev.index}):
            raise ValueError("a parameter's size or device is not that of its gradient or its moments")
        host, blocks = self._table(all_ps, all_grads, all_sts, sizes)
        with torch.cuda.device(dev):
            self._upload(host, blocks, dev)
            if self._slots is None:
                self._slots = torch.empty(_ADAMW_SLOTS, dtype=torch.float64, device=dev)
            stream = torch.cuda.current_stream(dev).cuda_stream
            table, entry_of = self._dev.data_ptr(), self._dev.data_ptr() + host.nbytes
            slots = norm = None
            if max_grad_norm is not None:
                norm = torch.empty((), dtype=torch.float32, device=dev)
                slots = self._slots.data_ptr()
                vitk.check(vitk.lib.vitk_adamw_norm(table, entry_of, int(blocks[-1]), float(max_grad_norm), slots, norm.data_ptr(),
                                                    stream), "adamw_norm")
            for group, t, first, cnt in spans:
                b1, b2 = group["betas"]
                block = int(host["block0"][first])
                vitk.check(vitk.lib.vitk_adamw_step(table, entry_of, block, int(blocks[first + cnt - 1]) - block, slots,
                                                    float(group["lr"]), float(b1), float(b2), float(group["eps"]),
                                                    float(group["weight_decay"]), t + 1, self.state_bits, self.seed, stream),
                           "adamw_step")
            for st in all_sts:
                st["step"] += 1
            # the parameters were written through raw pointers: graphs and operands that have kept them see a new version, and
            # the GEMM operands kept with them are renewed (one launch)
            torch.autograd.graph.increment_version(all_ps)
            vitk.ops.refresh_operands(all_ps)
        return norm

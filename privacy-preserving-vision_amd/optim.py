"""``ppv_amd.optim.Adam``: torch.optim.Adam with the whole parameter list updated by ONE hand-written kernel launch.

Reference use: the harness' optimisers, ``Image_Caption/train.py:92-101`` (``torch.optim.Adam(params=filter(lambda p: p.requires_grad,
encoder.parameters()), lr=encoder_lr)`` and the decoder's twin), stepped at ``train.py:318-321``.  Same constructor arguments, same
``param_groups`` / ``state`` layout (``step``, ``exp_avg``, ``exp_avg_sq`` per parameter, so ``state_dict()`` loads into
``torch.optim.Adam`` and back), same arithmetic as torch's fused kernel in f32 (``csrc/optim.hip``).  Not supported and refused loudly:
``amsgrad``, ``maximize``, ``capturable``, sparse or non-f32 gradients.  No CPU / stock-torch fallback: the HIP library does the step.

``ppv_amd.optim.AdamW``: torch.optim.AdamW (decoupled weight decay) the same way, with its moments in 32 or in 8 bits (``csrc/adamw.hip``)."""
import itertools
import operator
import struct

import numpy as np
import torch

from . import _lib

_CHUNK = 4096


class Adam(torch.optim.Optimizer):
    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0, amsgrad=False, *, maximize=False, capturable=False,
                 **ignored):
        if amsgrad or maximize or capturable:
            raise NotImplementedError("ppv_amd.optim.Adam: amsgrad / maximize / capturable are not implemented")
        if not 0.0 <= lr or not 0.0 <= eps or not 0.0 <= betas[0] < 1.0 or not 0.0 <= betas[1] < 1.0 or not 0.0 <= weight_decay:
            raise ValueError("ppv_amd.optim.Adam: invalid hyper-parameter")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, amsgrad=False, maximize=False,
                                      foreach=None, capturable=False, differentiable=False, fused=None))
        self._tables = {}                      # group index -> (key of data pointers, device descriptor table, total blocks)

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)    # new exp_avg / exp_avg_sq tensors: every cached descriptor table is stale
        self._tables = {}

    def __setstate__(self, state):
        super().__setstate__(state)
        self._tables = {}

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        self._tables = {}

    def _table(self, gi, ps):
        # the key holds EVERY pointer the records hold (parameter, gradient, both moments): a reloaded state or a re-allocated gradient
        # rebuilds the table instead of updating freed buffers
        key = tuple((p.data_ptr(), p.grad.data_ptr(), self.state[p]["exp_avg"].data_ptr(), self.state[p]["exp_avg_sq"].data_ptr()) for p in ps)
        hit = self._tables.get(gi)
        if hit is not None and hit[0] == key:
            return hit[1], hit[2]
        recs, blk = [], 0
        for p in ps:
            st = self.state[p]
            ptrs = (p.data_ptr(), p.grad.data_ptr(), st["exp_avg"].data_ptr(), st["exp_avg_sq"].data_ptr())
            vec = int(all(q % 16 == 0 for q in ptrs))
            recs.append(struct.pack("<QQQQqii", *ptrs, p.numel(), blk, vec))
            blk += (p.numel() + _CHUNK - 1) // _CHUNK
        desc = torch.from_numpy(np.frombuffer(b"".join(recs), dtype=np.uint8).copy()).to(ps[0].device)
        self._tables[gi] = (key, desc, blk)
        return desc, blk

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        L = _lib.lib()
        for gi, group in enumerate(self.param_groups):
            ps = [p for p in group["params"] if p.grad is not None]
            if not ps:
                continue
            dev = ps[0].device
            for p in ps:
                g = p.grad
                if (p.dtype != torch.float32 or g.dtype != torch.float32 or g.is_sparse or not p.is_contiguous() or not g.is_contiguous()
                        or p.device != dev or dev.type != "cuda"):
                    raise NotImplementedError("ppv_amd.optim.Adam: contiguous f32 parameters and gradients on one GPU only")
                st = self.state[p]
                if len(st) == 0:
                    st["step"] = torch.tensor(0.0, dtype=torch.float32)
                    st["exp_avg"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                    st["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.preserve_format)
            by_step = {}                       # parameters whose gradient was missing in some step keep their own count (as torch's do)
            for p in ps:
                by_step.setdefault(float(self.state[p]["step"]), []).append(p)
            b1, b2 = group["betas"]
            if len(by_step) > 1:               # split case: tables keyed by (group, slot), slots reused every step -> no growth with t
                for k in [k for k in self._tables if isinstance(k, tuple) and k[0] == gi and k[1] >= len(by_step)]:
                    del self._tables[k]
            for slot, (t, sub) in enumerate(sorted(by_step.items())):
                desc, blocks = self._table((gi, slot) if len(by_step) > 1 else gi, sub)
                n = t + 1.0
                _lib.check(L.ppv_adam_multi(desc.data_ptr(), len(sub), blocks, group["lr"], b1, b2, group["eps"], group["weight_decay"],
                                            1.0 - b1 ** n, 1.0 - b2 ** n, _lib.stream_ptr()), "ppv_adam_multi")
                # (written through addresses: autograd's check of saved tensors and the caches of weight layouts go by the version)
                torch.autograd.graph.increment_version([t for p in sub for t in (p, self.state[p]["exp_avg"], self.state[p]["exp_avg_sq"])])
                for p in sub:
                    self.state[p]["step"] += 1
        return loss


_CAPTURED = "ppv_amd.optim.AdamW: a step cannot be captured into a graph (its number is part of the launch)"


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW(params, lr, betas, eps, weight_decay) with every tensor of a group updated in one launch.

    ``state_bits=32``: ``exp_avg`` and ``exp_avg_sq`` in f32; ``state_dict()`` loads into torch.optim.AdamW and back.

    ``state_bits=8``: tensors of at least ``min_8bit_size`` elements keep 2 bytes of state per parameter instead of 8 (the smaller ones, biases
    and norm weights, stay in 32 bits): ``exp_avg`` and ``exp_avg_sq_root`` (the root of the second moment) as float8_e4m3fn, each with one
    f32 power-of-two scale per 256 consecutive elements (``exp_avg_scale``, ``exp_avg_sq_root_scale``; value = code * scale).  The new
    moments are computed in f32 and rounded stochastically, up with the probability of the upper neighbour's nearness: to the nearest, a second moment
    that moves by a thousandth per step would never leave its code.  The random numbers are a hash of ``seed``, the step, the tensor's
    place in the optimiser and the element's place in the tensor: the same run gives the same bits.

    Parameters and gradients are contiguous f32 tensors of one GPU per group; parameters without a gradient are left alone and keep their own
    step count (a float).  A step raises the versions of the parameters and moments that it wrote.  Refused: amsgrad, maximize, capturable, sparse
    gradients, tensors of one group that share memory (but for a parameter that is its own gradient), and a step inside a stream capture (the
    step's number is part of the launch, a replay would repeat it)."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, amsgrad=False, *, maximize=False, capturable=False,
                 state_bits=32, min_8bit_size=4096, seed=0):
        if amsgrad or maximize or capturable:
            raise NotImplementedError("ppv_amd.optim.AdamW: amsgrad / maximize / capturable are not implemented")
        if not 0.0 <= lr or not 0.0 <= eps or not 0.0 <= betas[0] < 1.0 or not 0.0 <= betas[1] < 1.0 or not 0.0 <= weight_decay:
            raise ValueError("ppv_amd.optim.AdamW: invalid hyper-parameter")
        if state_bits not in (8, 32):
            raise ValueError("ppv_amd.optim.AdamW: state_bits is 8 or 32")
        if min_8bit_size < 0:
            raise ValueError("ppv_amd.optim.AdamW: min_8bit_size >= 0")
        self.state_bits, self.min_8bit_size, self.seed = state_bits, min_8bit_size, int(seed)
        self._tables = {}                       # (group index, slot) -> (parameters, their moments, the native list of both)
        self._last = {}                         # group index -> what its last step was made of (_unchanged)
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, amsgrad=False, maximize=False,
                                      foreach=None, capturable=False, differentiable=False, fused=None))

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)
        for st in self.state.values():
            for k, x in st.items():            # own copies: the moments are updated in place, and the given state may be another optimiser's
                if k == "step":
                    st[k] = float(x)
                elif "exp_avg_scale" in st and not k.endswith("_scale"):
                    st[k] = x.to(torch.float8_e4m3fn)     # torch has cast the 8-bit values to the parameter's f32, where each of them exists
                else:
                    st[k] = x.clone(memory_format=torch.contiguous_format)
        self._tables, self._last = {}, {}

    def __getstate__(self):
        st = super().__getstate__()
        st.update(state_bits=self.state_bits, min_8bit_size=self.min_8bit_size, seed=self.seed)
        return st

    def __setstate__(self, state):
        super().__setstate__(state)
        for group in self.param_groups:        # (a state from before a group had these names)
            group.setdefault("amsgrad", False)
            group.setdefault("maximize", False)
        self._number()

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        ps = self.param_groups[-1]["params"]
        if len(set(ps)) != len(ps):             # (two records of one tensor in the one launch would race)
            del self.param_groups[-1]
            raise ValueError("ppv_amd.optim.AdamW: a parameter appears twice in a group")
        self._number()

    def _number(self):
        self._place = {p: i for i, p in enumerate(p for g in self.param_groups for p in g["params"])}
        self._tables, self._last = {}, {}

    def _init_state(self, p):
        st = self.state[p]
        st["step"] = 0.0
        if self.state_bits == 8 and p.numel() >= self.min_8bit_size:
            for k in ("exp_avg", "exp_avg_sq_root"):
                st[k] = torch.zeros(p.shape, dtype=torch.uint8, device=p.device).view(torch.float8_e4m3fn)
                st[k + "_scale"] = torch.zeros((p.numel() + 255) // 256, dtype=torch.float32, device=p.device)
        else:
            st["exp_avg"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
            st["exp_avg_sq"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)

    @staticmethod
    def _moments(st):
        """(m, v, scale of m, scale of v) of a parameter's state: which form it has is the state's own affair (it may have been loaded)."""
        if "exp_avg_scale" in st:
            return st["exp_avg"], st["exp_avg_sq_root"], st["exp_avg_scale"], st["exp_avg_sq_root_scale"]
        return st["exp_avg"], st["exp_avg_sq"], None, None

    def _list(self, slot, ps):
        """The native list of these parameters with their moments; kept while both are the same tensors."""
        sts = [self.state[p] for p in ps]
        held = [t for st in sts for t in self._moments(st)]
        hit = self._tables.get(slot)
        if hit is not None and len(hit[0]) == len(ps) and all(map(operator.is_, hit[0], ps)) and all(map(operator.is_, hit[1], held)):
            return hit[2]
        for p, (m, v, ms, vs) in zip(ps, zip(*[iter(held)] * 4)):
            n, kind = p.numel(), torch.float32 if ms is None else torch.float8_e4m3fn
            if not (all(t.device == p.device and t.is_contiguous() and t.numel() == n and t.dtype == kind for t in (m, v)) and (ms is None or all(
                    t.device == p.device and t.is_contiguous() and t.numel() == (n + 255) // 256 and t.dtype == torch.float32 for t in (ms, vs)))):
                raise ValueError("ppv_amd.optim.AdamW: a parameter's state does not belong to it (type, size, device or layout)")
        native = _lib.torch_ops().AdamWList(ps, held[0::4], held[1::4], held[2::4], held[3::4], [self._place[p] & 0xFFFFFFFF for p in ps])
        self._tables[slot] = (ps, held, native)
        return native

    def _unchanged(self, gi, group):
        """What the group's last step was made of, if all of it is as it was: the parameters, every state and every entry of it (moments and the common
        step number), which parameters have gradients.  None if not, or if they had several step numbers: then the step starts from the states.
        (Identities only, no look-up per parameter: 333 tensors took 460 us of host time from the states, 90 so.)"""
        last = self._last.get(gi)
        if last is None:
            return None
        params, states, sts, entries, _, native = last
        same = lambda a, b: len(a) == len(b) and all(map(operator.is_, a, b))
        if (same(params, group["params"]) and same(states, self.state.values()) and
                same(list(itertools.chain.from_iterable(map(dict.values, sts))), entries) and native.complete()):
            return last
        return None

    def _remember(self, gi, group, ps, native):
        sts = [self.state[p] for p in ps]
        native.without([p for p in group["params"] if p.grad is None])
        items = [kv for st in sts for kv in st.items()]
        self._last[gi] = (list(group["params"]), list(self.state.values()), sts, [v for _, v in items],
                          [i for i, (k, _) in enumerate(items) if k == "step"], native)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for gi, group in enumerate(self.param_groups):
            if group["amsgrad"] or group["maximize"]:           # (a group's own, or a loaded one's)
                raise NotImplementedError("ppv_amd.optim.AdamW: amsgrad / maximize are not implemented")
            b1, b2 = group["betas"]
            hyper = lambda n: (float(group["lr"]), b1, b2, group["eps"], group["weight_decay"], n, self.seed & 0xFFFFFFFF)
            last = self._unchanged(gi, group)
            if last is not None:
                _, _, sts, entries, at, native = last
                if torch.cuda.is_current_stream_capturing():
                    raise RuntimeError(_CAPTURED)
                n = entries[at[0]] + 1.0
                native.step(*hyper(n))
                for st, i in zip(sts, at):
                    st["step"] = entries[i] = n
                continue
            self._last.pop(gi, None)
            ps = [p for p in group["params"] if p.grad is not None]
            if not ps:
                continue
            if ps[0].device.type != "cuda":
                raise NotImplementedError("ppv_amd.optim.AdamW: contiguous f32 parameters and gradients on one GPU only")
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError(_CAPTURED)
            for p in ps:
                if not self.state[p]:
                    self._init_state(p)
            by_step = {}                       # parameters whose gradient was missing in some step keep their own count
            for p in ps:
                by_step.setdefault(float(self.state[p]["step"]), []).append(p)
            for k in [k for k in self._tables if k[0] == gi and k[1] >= len(by_step)]:
                del self._tables[k]
            for slot, (t, sub) in enumerate(sorted(by_step.items())):
                native, n = self._list((gi, slot), sub), t + 1.0
                native.step(*hyper(n))
                for p in sub:
                    self.state[p]["step"] = n
            if len(by_step) == 1:
                self._remember(gi, group, ps, native)
        return loss

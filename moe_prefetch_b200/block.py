"""The operators around an expert layer: routing rules, the norms before and
after it with its gate and residual, and low-rank adapters of many requests.

``Routing``, ``BlockNorm`` and ``AdapterSet`` hold what a model keeps between
calls (the rule, the norm weights, the adapters laid out for the kernels) and
are called on device tensors.  ``MoeStack.set_routing`` gives a layer a routing
rule, and ``MoeStack.block_forward`` runs a whole layer with all three.

They are for inference: no call records a gradient.  Every call takes its work to the tensors' device, on that device's current
stream or on ``stream``; nothing waits for the host, and the calls can be
captured in a CUDA graph.  With ``stream`` the caller orders it after the
producers of the inputs; the outputs are allocated for that stream.

An output given with ``out`` may be an input where the call says so (the same
memory with the same type and strides), and may lie between the rows of other
tensors; any other overlap is a MoeError.
"""
import ctypes as C

import torch

from . import _lib
from ._lib import MoeAdapters, MoeNorm, MoeRouteCfg, check

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
SCORES = {"softmax": 0, "sigmoid": 1}
SCORE_MASKED = 0x100
ACTS = {"none": 0, "sigmoid": 1}
_ROWS = torch.contiguous_format
GATE_NONE, GATE_TOKEN, GATE_CHANNEL, GATE_FULL = 0, 1, 2, 3


# The current stream's handle without a Stream object (torch.cuda.current_stream
# takes 2 us of a call's 9), where this torch has it.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _rows(t, name, width, dtypes=DTYPES):
    """Check a [n, width] device tensor with contiguous rows; its row stride."""
    shape = t.shape
    if len(shape) != 2 or shape[1] != width:
        raise ValueError(f"{name} must be [n, {width}], got {tuple(shape)}")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} has type {t.dtype}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be on a CUDA device")
    ld, inner = t.stride()
    if inner != 1 and width > 1:
        raise ValueError(f"{name}: the elements of a row must be contiguous")
    if shape[0] <= 1:
        return width
    if ld < width:
        raise ValueError(f"{name}: rows overlap (row stride {ld})")
    return ld


def _vector(t, name, n, dtype, device):
    if t.shape != (n,) or t.dtype != dtype or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} [{n}] on {device}, got {t.dtype} {tuple(t.shape)} "
                         f"on {t.device}")
    return t.data_ptr()


def _same_device(device, **tensors):
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name} is on {t.device}, expected {device}")


def _on_stream(call, stream, tensors):
    """call() with `stream` current, which its device's allocator then knows
    the tensors are used on."""
    for t in tensors:
        if t is not None and t.is_cuda and t.device != stream.device:
            raise ValueError(f"the stream is on {stream.device}, a tensor on {t.device}")
    with torch.cuda.stream(stream):
        out = call()
    for t in tensors:
        if t is not None:
            t.record_stream(stream)
    return out


# the current device's index (a call on tensors of another one enters it first)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


class Routing:
    """A routing rule (moe_route_cfg): scores softmax or sigmoid, a bias for
    balance that decides who is chosen but never the weight, n_group groups of
    which the topk_group best are kept (by their largest value, or with
    group_top 2 by the sum of their two largest), the k best experts, weights
    divided by their sum (renorm) and multiplied by scale.  With masked a logit of
    -inf switches its expert off for that token: it is chosen last, whatever its
    bias (without, its score is 0 and the bias may choose it, with weight 0).

    ``routing(logits)`` -> ids int32 [n, k], w fp32 [n, k].  Ties go to the
    lower expert; a logit of -inf has score 0, and with a bias of -inf an expert
    is chosen last.  The bias tensor's memory is read at every call, so that a
    change of its values in place is seen (MoeStack.set_routing copies it);
    other memory that the tensor is given later (``bias.data = ...``) is not."""

    def __init__(self, n_expert, k, score="softmax", bias=None, n_group=1, topk_group=None, group_top=1,
                 renorm=True, scale=1.0, masked=False):
        if score not in SCORES:
            raise ValueError(f"unknown score {score!r}")
        self.lib = _lib.load()
        self.n_expert, self.k = n_expert, k
        self.cfg = MoeRouteCfg(n_expert, k, SCORES[score] | (SCORE_MASKED if masked else 0), n_group,
                               n_group if topk_group is None else topk_group, group_top, int(bool(renorm)), scale)
        check(self.lib.moe_route(C.byref(self.cfg), None, 0, n_expert, 0, None, None, None, None), None, "moe_route")
        if bias is not None and (bias.shape != (n_expert,) or bias.dtype != torch.float32):
            raise ValueError(f"bias must be fp32 [{n_expert}], got {bias.dtype} {tuple(bias.shape)}")
        self.bias = None if bias is None else bias.detach()   # (keeps the memory whose address is used)
        # (the bias of a strided tensor is gathered by every call)
        self.bias_ptr = None if bias is None or not bias.is_contiguous() else bias.data_ptr()
        self.cfg_ref = C.byref(self.cfg)

    def __call__(self, logits, out=None, stream=None):
        """logits [n, n_expert] (fp32, bf16 or fp16) -> (ids, w); out: the
        (ids, w) to write."""
        if stream is not None:
            return _on_stream(lambda: self(logits, out), stream, (logits, self.bias, *(out or ())))
        index = logits.get_device()
        if index >= 0 and index != _current_device():
            with torch.cuda.device(index):
                return self(logits, out)
        ld = _rows(logits, "logits", self.n_expert)
        device, n, k = logits.device, logits.shape[0], self.k
        bias, bias_ptr = self.bias, self.bias_ptr
        if bias is not None:
            if bias.device != device:
                raise ValueError(f"the bias is on {bias.device}, the logits are on {device}")
            if bias_ptr is None:
                bias = bias.contiguous()
                bias_ptr = bias.data_ptr()
        if out is None:
            ids = torch.empty(n, k, dtype=torch.int32, device=device)
            w = torch.empty(n, k, dtype=torch.float32, device=device)
        else:
            ids, w = out
            if (ids.shape != (n, k) or w.shape != (n, k) or ids.dtype != torch.int32 or w.dtype != torch.float32
                    or not ids.is_contiguous() or not w.is_contiguous()):
                raise ValueError(f"out must be contiguous int32 and fp32 [{n}, {k}]")
            _same_device(device, ids=ids, w=w)
        rc = self.lib.moe_route(self.cfg_ref, logits.data_ptr(), DTYPES[logits.dtype], ld, n, bias_ptr,
                                ids.data_ptr(), w.data_ptr(), _raw_stream(index))
        if rc:
            check(rc, None, "moe_route")
        return ids, w


class BlockNorm:
    """The norms around a block of width n_embd (moe_norm):

        z  = y / sqrt(mean(y^2) + eps) * (post + weight_offset)    (z = y without post)
        r' = r + scale * gate_act(gate) * z
        x  = r' / sqrt(mean(r'^2) + eps) * (pre + weight_offset)

    post, pre: fp32 [n_embd] weights, or None (post None: no norm after the
    block; pre None: no x; pre True: x with weight 1); their memory is read at
    every call, as a Routing's bias is.  ``norm(r, y)`` and
    ``norm.combine(r, y_rows, pos, w)`` return (r', x)."""

    def __init__(self, n_embd, post=None, pre=None, gate_act="none", scale=1.0, eps=1e-6, weight_offset=0.0):
        if gate_act not in ACTS:
            raise ValueError(f"unknown gate activation {gate_act!r}")
        self.lib = _lib.load()
        self.n_embd = n_embd
        self.with_x = pre is not None and pre is not False
        self.post = None if post is None else post.detach()
        self.pre = pre.detach() if isinstance(pre, torch.Tensor) else None
        for name, t in (("post", self.post), ("pre", self.pre)):
            if t is not None and (t.shape != (n_embd,) or t.dtype != torch.float32 or not t.is_contiguous()):
                raise ValueError(f"{name} must be a contiguous fp32 [{n_embd}]")
        self.device = next((t.device for t in (self.post, self.pre) if t is not None), None)
        if None not in (self.post, self.pre) and self.post.device != self.pre.device:
            raise ValueError(f"post is on {self.post.device}, pre on {self.pre.device}")
        self.nm = MoeNorm(n_embd, GATE_NONE, ACTS[gate_act], scale, eps, weight_offset,
                          None if self.post is None else self.post.data_ptr(),
                          None if self.pre is None else self.pre.data_ptr(), None, 0)
        self.nm_ref = C.byref(self.nm)
        check(self.lib.moe_block_norm(self.nm_ref, None, 0, n_embd, None, 0, n_embd, None, n_embd, None, n_embd,
                                      0, None), None, "moe_block_norm")

    def with_gate(self, gate, n, dtype, device):
        """The moe_norm of one call; gate None, [n, 1] (per row), [n_embd] (per
        channel, fp32) or [n, n_embd]."""
        if gate is None:
            return self.nm
        if gate.device != device:
            raise ValueError(f"the gate is on {gate.device}, expected {device}")
        nm = MoeNorm.from_buffer_copy(self.nm)   # a call's own: calls may run at the same time
        nm.gate = gate.data_ptr()
        if gate.shape == (self.n_embd,):
            _vector(gate, "a gate per channel", self.n_embd, torch.float32, device)
            nm.gate_kind = GATE_CHANNEL
        elif gate.shape == (n, 1):
            if gate.dtype != dtype:
                raise ValueError(f"the gate has type {gate.dtype}, expected {dtype}")
            nm.gate_kind, nm.ld_gate = GATE_TOKEN, gate.stride(0) if n > 1 else 1
        else:
            if gate.dim() != 2 or gate.shape[0] != n or gate.dtype != dtype:
                raise ValueError(f"the gate must be {dtype} [{n}, 1] or [{n}, {self.n_embd}], or fp32 "
                                 f"[{self.n_embd}], got {gate.dtype} {tuple(gate.shape)}")
            nm.ld_gate = _rows(gate, "gate", self.n_embd)
            nm.gate_kind = GATE_FULL
        return nm

    def _check_out(self, r, dtype, out):
        n, h = r.shape
        ro, x = out
        if (x is not None) != self.with_x or ro is None and x is None:
            raise ValueError("out must be (r', x), with None for x without a second norm")
        lro = ldx = h
        if ro is not None:
            lro = _rows(ro, "out r'", h, (r.dtype,))
        if x is not None:
            ldx = _rows(x, "out x", h, (dtype,))
        for t in (ro, x):
            if t is not None and t.shape[0] != n:
                raise ValueError(f"out must have {n} rows")
        _same_device(r.device, r_out=ro, x=x)
        return ro, x, lro, ldx

    def __call__(self, r, y=None, gate=None, out=None, stream=None):
        """r [n, n_embd] the residual, fp32 or y's type; y the block's output
        (None: r' = r, the norm of a first block); out: (r', x) to write, r'
        may be None (not wanted); each may be r, y or a full gate, but not the
        other."""
        if stream is not None:
            return _on_stream(lambda: self(r, y, gate, out), stream,
                              (r, y, gate, self.post, self.pre, *(out or ())))
        index = r.get_device()
        if index >= 0 and index != _current_device():
            with torch.cuda.device(index):
                return self(r, y, gate, out)
        ld_r = _rows(r, "r", self.n_embd)
        device, n = r.device, r.shape[0]
        dtype, ld_y, y_ptr = r.dtype, self.n_embd, None
        if y is not None:
            ld_y = _rows(y, "y", self.n_embd)
            dtype, y_ptr = y.dtype, y.data_ptr()
            if y.shape[0] != n:
                raise ValueError(f"y has {y.shape[0]} rows, r has {n}")
            if y.device != device:
                raise ValueError(f"y is on {y.device}, expected {device}")
        elif out is not None and out[1] is not None:
            dtype = out[1].dtype
        nm = self.nm_ref if gate is None else C.byref(self.with_gate(gate, n, dtype, device))
        if self.device is not None and self.device != device:
            raise ValueError(f"the norm's weights are on {self.device}, expected {device}")
        if out is None:
            lro = ldx = self.n_embd
            ro = torch.empty_like(r, memory_format=_ROWS)
            x = torch.empty_like(r if y is None else y, memory_format=_ROWS) if self.with_x else None
        else:
            ro, x, lro, ldx = self._check_out(r, dtype, out)
        rc = self.lib.moe_block_norm(nm, r.data_ptr(), DTYPES[r.dtype], ld_r, y_ptr, DTYPES[dtype], ld_y,
                                     None if ro is None else ro.data_ptr(), lro,
                                     None if x is None else x.data_ptr(), ldx, n, _raw_stream(index))
        if rc:
            check(rc, None, "moe_block_norm")
        return ro, x

    def combine(self, r, y_rows, pos, w, add=None, gate=None, out=None, stream=None):
        """The same with y the combine of an expert layer's rows, y[t] = sum_j
        w[t, j] * y_rows[pos[t, j]] (+ add[t]); fp32, pos int32.  A pos
        outside y_rows adds nothing, whatever its weight.  out: each may be r,
        add or a full gate, but not the other."""
        if stream is not None:
            return _on_stream(lambda: self.combine(r, y_rows, pos, w, add, gate, out), stream,
                              (r, y_rows, pos, w, add, gate, self.post, self.pre, *(out or ())))
        index = r.get_device()
        if index >= 0 and index != _current_device():
            with torch.cuda.device(index):
                return self.combine(r, y_rows, pos, w, add, gate, out)
        f32 = (torch.float32,)
        h = self.n_embd
        ld_r, ld_rows = _rows(r, "r", h, f32), _rows(y_rows, "y_rows", h, f32)
        device, n = r.device, r.shape[0]
        shape = pos.shape
        k = shape[1] if len(shape) == 2 else 0
        if (k == 0 or shape[0] != n or w.shape != shape or pos.dtype != torch.int32 or w.dtype != torch.float32
                or not pos.is_contiguous() or not w.is_contiguous()):
            raise ValueError(f"pos and w must be contiguous int32 and fp32 [{n}, k]")
        if add is not None and (add.shape != (n, h) or add.dtype != torch.float32 or not add.is_contiguous()):
            raise ValueError(f"add must be a contiguous fp32 [{n}, {h}]")
        if y_rows.device != device or pos.device != device or w.device != device or (add is not None and add.device != device):
            raise ValueError(f"r is on {device}, and y_rows, pos, w and add must be")
        nm = self.nm_ref if gate is None else C.byref(self.with_gate(gate, n, torch.float32, device))
        if self.device is not None and self.device != device:
            raise ValueError(f"the norm's weights are on {self.device}, expected {device}")
        if out is None:
            lro = ldx = h
            ro = torch.empty_like(r, memory_format=_ROWS)
            x = torch.empty_like(r, memory_format=_ROWS) if self.with_x else None
        else:
            ro, x, lro, ldx = self._check_out(r, torch.float32, out)
        rc = self.lib.moe_combine_norm(nm, r.data_ptr(), ld_r, y_rows.data_ptr(), ld_rows, y_rows.shape[0],
                                       pos.data_ptr(), w.data_ptr(), k, None if add is None else add.data_ptr(),
                                       None if ro is None else ro.data_ptr(), lro,
                                       None if x is None else x.data_ptr(), ldx, n, _raw_stream(index))
        if rc:
            check(rc, None, "moe_combine_norm")
        return ro, x


class AdapterSet:
    """Low-rank adapters of one projection (moe_adapters): a [n, r, n_in] and
    b [n, n_out, r] in bf16 or fp16 on the device, or lists of n per-adapter
    [r_i, n_in] / [n_out, r_i].  scale: a number, or fp32 [n] (alpha / r in the
    usual parametrisation); rank: int32 [n] ranks in use, where they differ.

    ``adapters(x, ids, y)`` -> y[t] + scale[i] * b[i] (a[i] x[t]), i = ids[t];
    a row with id -1 (or any id outside the set) keeps y[t].  The weights are
    laid out once, here, on the current stream; a later change of a or b is not
    seen.  How many bits of x and of A x the products use stands at
    moe_adapters_apply."""

    MAX_RANK = 128

    def __init__(self, a, b, scale=1.0, rank=None):
        self.lib = _lib.load()
        if isinstance(a, (list, tuple)):
            if not a or len(a) != len(b) or rank is not None:
                raise ValueError("lists of adapters: one a and one b each, and no rank")
            ranks = [t.shape[0] for t in a]
            if [t.shape[-1] for t in b] != ranks:
                raise ValueError(f"ranks {ranks} of a, {[t.shape[-1] for t in b]} of b")
            a = torch.stack([torch.nn.functional.pad(t, (0, 0, 0, max(ranks) - t.shape[0])) for t in a])
            b = torch.stack([torch.nn.functional.pad(t, (0, max(ranks) - t.shape[1])) for t in b])
            rank = torch.tensor(ranks, dtype=torch.int32, device=a.device)
        if a.dim() != 3 or b.dim() != 3 or a.shape[0] != b.shape[0] or a.shape[1] != b.shape[2] or 0 in a.shape + b.shape:
            raise ValueError(f"a must be [n, r, n_in] and b [n, n_out, r], got {tuple(a.shape)} and {tuple(b.shape)}")
        if a.dtype != b.dtype or a.dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"a and b must both be bf16 or fp16, got {a.dtype} and {b.dtype}")
        if not a.is_cuda or a.device != b.device:
            raise ValueError(f"a and b must be on one CUDA device, got {a.device} and {b.device}")
        self.n, r, self.n_in = a.shape
        self.n_out = b.shape[1]
        if r > self.MAX_RANK:
            raise ValueError(f"rank {r} is above {self.MAX_RANK}")
        self.dtype, self.device = a.dtype, a.device
        pr, pc = -r % 8, -self.n_in % 8
        # rank to a multiple of 8 and n_in to a multiple of 8, with zeros
        self.a = torch.nn.functional.pad(a.detach(), (0, pc, 0, pr)) if pr or pc else a.detach().clone(
            memory_format=torch.contiguous_format)
        self.b = torch.nn.functional.pad(b.detach(), (0, pr)) if pr else b.detach().clone(
            memory_format=torch.contiguous_format)
        if not isinstance(scale, torch.Tensor):
            scale = torch.full((self.n,), float(scale), device=self.device)
        elif scale.shape != (self.n,):
            raise ValueError(f"scale must be a number or [{self.n}], got {tuple(scale.shape)}")
        self.scale = scale.to(device=self.device, dtype=torch.float32, copy=True)
        if rank is None and pr:
            rank = torch.full((self.n,), r, dtype=torch.int32, device=self.device)
        elif rank is not None and tuple(rank.shape) != (self.n,):
            raise ValueError(f"rank must be [{self.n}], got {tuple(rank.shape)}")
        self.rank = None if rank is None else rank.to(device=self.device, dtype=torch.int32, copy=True).clamp_(0, r)
        self.st = MoeAdapters(self.a.data_ptr(), self.b.data_ptr(), self.scale.data_ptr(),
                              None if self.rank is None else self.rank.data_ptr(), self.n, r + pr, self.n_in,
                              self.n_out, DTYPES[self.dtype], self.n_in + pc)
        self.st_ref, self.index = C.byref(self.st), self.a.get_device()
        check(self.lib.moe_adapters_apply(self.st_ref, None, None, self.st.dtype, self.n_in, None, 0, None,
                                          self.st.dtype, self.n_out, 0, None), None, "moe_adapters_apply")

    def check_ids(self, ids, n):
        _vector(ids, "ids", n, torch.int32, self.device)

    def __call__(self, x, ids, y=None, out=None, out_dtype=None, stream=None):
        """x [n, n_in] fp32 or the weights' type; ids int32 [n]; y [n, n_out]
        (None: zeros); out: where to write, may be y.  y and out are fp32, or
        the weights' type where x is.  out_dtype: the output's type without y
        and out (default x's)."""
        if stream is not None:
            return _on_stream(lambda: self(x, ids, y, out, out_dtype), stream,
                              (x, ids, y, out, self.a, self.b, self.scale, self.rank))
        index = self.index
        if index != _current_device():
            with torch.cuda.device(index):
                return self(x, ids, y, out, out_dtype)
        device = self.device
        ld_x = _rows(x, "x", self.n_in)
        n = x.shape[0]
        if x.device != device:
            raise ValueError(f"x is on {x.device}, expected {device}")
        ids_ptr = _vector(ids, "ids", n, torch.int32, device)
        ld_y = ld_o = self.n_out
        y_ptr = None
        if y is not None:
            ld_y = _rows(y, "y", self.n_out)
            y_ptr = y.data_ptr()
            if y.shape[0] != n or y.device != device:
                raise ValueError(f"y has {y.shape[0]} rows on {y.device}, expected {n} on {device}")
        if out is None:
            out = (torch.empty(n, self.n_out, dtype=out_dtype or x.dtype, device=device) if y is None
                   else torch.empty_like(y, memory_format=_ROWS))
        else:
            ld_o = _rows(out, "out", self.n_out)
            if out.shape[0] != n or out.device != device or (y is not None and out.dtype != y.dtype):
                raise ValueError("out must have x's rows and device and y's type")
        if out.dtype not in DTYPES:
            raise ValueError(f"out has type {out.dtype}")
        rc = self.lib.moe_adapters_apply(self.st_ref, ids_ptr, x.data_ptr(), DTYPES[x.dtype], ld_x, y_ptr, ld_y,
                                         out.data_ptr(), DTYPES[out.dtype], ld_o, n, _raw_stream(index))
        if rc:
            check(rc, None, "moe_adapters_apply")
        return out

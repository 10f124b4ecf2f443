"""Operators of a learned prior over a texture's symbols, on torch tensors (the C ABI of include/ntc_ops.h).

    token_logprobs(logits, tokens, top=0)     log probabilities of given tokens, entropy, the best alternatives; differentiable
    AdamW(params, state_bits=32 or 8).step()  one step over many tensors
    fp8_quantize(x), fp8_matmul(a, b)         8-bit floating point with a power-of-two scale for each block of 128
    fp8_linear(x, w)                          a layer in it, for training or, with weights laid out once, for inference

Tensors are on the GPU; work is enqueued on torch's current stream and nothing waits. Arguments that an operator does not
take raise ValueError, errors of the runtime RuntimeError. There is no fallback: the kernels are libntc_hip.so's.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import NamedTuple, Optional

import numpy as np
import torch

from . import trainer

MAX_TOP, STATE_BLOCK, CHUNK = 32, 256, 4096
_CODE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_FP8 = 3
_P, _L, _I = C.c_void_p, C.c_int64, C.c_int32


class LogprobsDesc(C.Structure):
    _fields_ = [("logits", _P), ("tokens", _P), ("rows", _L), ("inner_rows", _L), ("V", _L), ("outer_stride", _L), ("inner_stride", _L),
                ("token_outer_stride", _L), ("token_inner_stride", _L), ("ignore_index", _L), ("dtype", _I), ("token_bytes", _I), ("top", _I),
                ("temperature", C.c_float), ("logprob", _P), ("entropy", _P), ("stats", _P), ("top_ids", _P), ("top_logprobs", _P),
                ("workspace", _P), ("g_logprob", _P), ("g_entropy", _P), ("g_top", _P), ("dlogits", _P)]


class AdamwDesc(C.Structure):
    _fields_ = [("tensors", _P), ("chunk_tensor", _P), ("first_chunk", _P), ("grads", _P), ("grad_types", _P), ("steps", _P), ("n", _L),
                ("exp_avg", _P), ("exp_avg_sq", _P), ("exp_avg_exp", _P), ("exp_avg_sq_exp", _P), ("master", _P), ("lr", C.c_double),
                ("beta1", C.c_double), ("beta2", C.c_double), ("eps", C.c_double), ("weight_decay", C.c_double), ("seed", C.c_uint64),
                ("calls", C.c_uint32), ("state_bits", _I)]


class QuantizeDesc(C.Structure):
    _fields_ = [("x", _P), ("R", _L), ("K", _L), ("row_stride", _L), ("dtype", _I), ("block_rows", _I), ("codes", _P), ("exps", _P), ("codes_t", _P),
                ("exps_t", _P)]


class MatmulDesc(C.Structure):
    _fields_ = [("a", _P), ("a_exps", _P), ("b", _P), ("b_exps", _P), ("c", _P), ("workspace", _P), ("M", _L), ("N", _L), ("K", _L), ("a_stride", _L),
                ("ldc", _L), ("a_type", _I), ("a_block_rows", _I), ("b_block_rows", _I), ("c_type", _I)]


_TENSOR = np.dtype([("param", np.uint64), ("numel", np.int64), ("state_offset", np.int64), ("param_type", np.int32), ("first_chunk", np.int32)])
_lib = None


def library() -> C.CDLL:
    global _lib
    if _lib is None:
        lib = trainer.library()
        tail = [_P, C.c_char_p, C.c_size_t]
        sig = {
            "ntc_op_token_logprobs_workspace": (C.c_size_t, [_L, _L, _I, _I]),
            "ntc_op_token_logprobs": (C.c_int, [_P] + tail),
            "ntc_op_token_logprobs_backward": (C.c_int, [_P] + tail),
            "ntc_op_adamw": (C.c_int, [_P] + tail),
            "ntc_op_adamw_moments": (C.c_int, [_P, _P, _P, _P, _L, _P, _P] + tail),
            "ntc_op_adamw_encode": (C.c_int, [_P, _P, _L, _P, _P, _P, _P] + tail),
            "ntc_op_fp8_quantize": (C.c_int, [_P] + tail),
            "ntc_op_fp8_matmul_workspace": (C.c_size_t, [_L, _L, _L]),
            "ntc_op_fp8_matmul": (C.c_int, [_P] + tail),
            "ntc_op_fp8_matmul_float_rows": (_L, []),
        }
        for name, (res, args) in sig.items():
            fn = getattr(lib, name)
            fn.restype, fn.argtypes = res, args
        _lib = lib
    return _lib


def _call(device: torch.device, fn, *args) -> None:
    """One entry point on the device's current stream; its refusal as ValueError, the runtime's as RuntimeError."""
    why = C.create_string_buffer(256)
    if torch.cuda.current_device() == device.index:
        rc = fn(*args, torch.cuda.current_stream(device).cuda_stream, why, 256)
    else:
        with torch.cuda.device(device):
            rc = fn(*args, torch.cuda.current_stream(device).cuda_stream, why, 256)
    if rc:
        raise (ValueError if rc == 1 else RuntimeError)(why.value.decode())


def _on_gpu(name: str, t, types=None) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a tensor on the GPU")
    if types is not None and t.dtype not in types:
        raise ValueError(f"{name} is {t.dtype}; it can be {', '.join(str(x) for x in types)}")
    return t


# ---------------------------------------------------------------- token log probabilities
class TokenLogprobs(NamedTuple):
    """What token_logprobs returns: in nats, 32-bit floats, in the tokens' shape (and one more axis for the alternatives)."""
    logprob: torch.Tensor
    entropy: torch.Tensor
    top_ids: Optional[torch.Tensor] = None
    top_logprobs: Optional[torch.Tensor] = None


def _rows(t: torch.Tensor, lead: tuple, name: str):
    """(rows, rows of the inner axis, outer stride, inner stride) of a tensor whose leading axes are `lead`."""
    strides = t.stride()[:len(lead)]
    if len(lead) == 0:
        return 1, 1, 0, 0
    if len(lead) == 1:
        return lead[0], max(1, lead[0]), 0, strides[0]
    if len(lead) > 2:
        try:
            t = t.view(-1, *t.shape[len(lead) - 1:])
        except RuntimeError:
            raise ValueError(f"the rows of {name} must lie at two strides at most") from None
        return _rows(t, tuple(t.shape[:2]), name)
    return lead[0] * lead[1], max(1, lead[1]), strides[0], strides[1]


def _logprobs_desc(logits, tokens, top, temperature, ignore_index) -> LogprobsDesc:
    lead = tuple(logits.shape[:-1])
    d = LogprobsDesc()
    d.logits, d.tokens = logits.data_ptr(), tokens.data_ptr()
    d.rows, d.inner_rows, d.outer_stride, d.inner_stride = _rows(logits, lead, "logits")
    _, _, d.token_outer_stride, d.token_inner_stride = _rows(tokens, lead, "tokens")
    d.V, d.ignore_index, d.dtype, d.token_bytes = logits.shape[-1], ignore_index, _CODE[logits.dtype], tokens.element_size()
    d.top, d.temperature = top, temperature
    return d


def _logprobs_forward(logits, tokens, top, temperature, ignore_index):
    d = _logprobs_desc(logits, tokens, top, temperature, ignore_index)
    shape, new = tokens.shape, logits.new_empty
    logprob, entropy = new(shape, dtype=torch.float32), new(shape, dtype=torch.float32)
    stats = new((*shape, 2), dtype=torch.float32)
    d.logprob, d.entropy, d.stats = logprob.data_ptr(), entropy.data_ptr(), stats.data_ptr()
    ids = top_logprobs = None
    if top:
        ids, top_logprobs = new((*shape, top), dtype=torch.int64), new((*shape, top), dtype=torch.float32)
        d.top_ids, d.top_logprobs = ids.data_ptr(), top_logprobs.data_ptr()
    size = library().ntc_op_token_logprobs_workspace(d.rows, d.V, d.dtype, top)
    work = new(size, dtype=torch.uint8) if size else None
    d.workspace = None if work is None else work.data_ptr()
    _call(logits.device, library().ntc_op_token_logprobs, C.byref(d))
    return logprob, entropy, ids, top_logprobs, stats


class _TokenLogprobsGrad(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, top, temperature, ignore_index):
        logprob, entropy, ids, top_logprobs, stats = _logprobs_forward(logits, tokens, top, temperature, ignore_index)
        ctx.args = top, temperature, ignore_index
        ctx.save_for_backward(logits, tokens, entropy, stats, ids)
        ctx.set_materialize_grads(False)
        if ids is not None:
            ctx.mark_non_differentiable(ids)
        return logprob, entropy, ids, top_logprobs

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_logprob, g_entropy, _, g_top):
        logits, tokens, entropy, stats, ids = ctx.saved_tensors
        if g_logprob is None and g_entropy is None and g_top is None:
            return None, None, None, None, None
        d = _logprobs_desc(logits, tokens, *ctx.args)
        grads = [None if g is None else g.contiguous() for g in (g_logprob, g_entropy, g_top)]
        d.g_logprob, d.g_entropy, d.g_top = (None if g is None else g.data_ptr() for g in grads)
        dlogits = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        d.entropy, d.stats, d.dlogits = entropy.data_ptr(), stats.data_ptr(), dlogits.data_ptr()
        d.top_ids = None if ids is None else ids.data_ptr()
        _call(logits.device, library().ntc_op_token_logprobs_backward, C.byref(d))
        return dlogits, None, None, None, None


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0, temperature: float = 1.0, ignore_index: int = -100) -> TokenLogprobs:
    """Log probabilities of `tokens` under softmax(logits / temperature), the distribution's entropy, and its `top` (at most 32)
    most probable symbols in descending order, equal ones by ascending index.

    logits [.., V]: float32, bfloat16 or float16, a row's values contiguous, rows at any two strides (a [batch, time, V] tensor's
    [:, :-1] as it lies). tokens [..]: int32 or int64. A token equal to ignore_index has logprob 0 and no gradient;
    another one outside [0, V) has logprob NaN. -inf masks a symbol; a row with nothing left has log probabilities -inf, entropy 0
    and gradient 0; a NaN or +inf makes its row's results NaN (ids then order NaN as -inf). logprob, entropy and top_logprobs are
    differentiable in logits (once); log probabilities and sums are 32-bit, dlogits is rounded once to the logits' type.
    """
    _on_gpu("logits", logits, (torch.float32, torch.bfloat16, torch.float16))
    _on_gpu("tokens", tokens, (torch.int64, torch.int32))
    if logits.dim() < 1 or tokens.shape != logits.shape[:-1] or tokens.device != logits.device:
        raise ValueError(f"tokens {tuple(tokens.shape)} must have the shape of logits {tuple(logits.shape)} without its last axis, on its device")
    V = logits.shape[-1]
    if V < 1 or (V > 1 and logits.stride(-1) != 1):
        raise ValueError("a row of logits must hold at least one value, contiguous")
    if not 0 <= top <= min(MAX_TOP, V):
        raise ValueError(f"top is 0 to {min(MAX_TOP, V)}, not {top}")
    if not 0 < temperature < 3e38:
        raise ValueError(f"temperature must be positive and finite, not {temperature}")
    if tokens.dim() > 2:
        tokens = tokens.contiguous()
    if logits.requires_grad and torch.is_grad_enabled():
        return TokenLogprobs(*_TokenLogprobsGrad.apply(logits, tokens, top, temperature, ignore_index))
    return TokenLogprobs(*_logprobs_forward(logits, tokens, top, temperature, ignore_index)[:4])


# ---------------------------------------------------------------- AdamW
class AdamW:
    """AdamW over many tensors in few launches, its state in 32 bits or in 8.

    params: contiguous GPU tensors (float32, bfloat16, float16, mixed as they come) of one device; they are updated in place. With
    `master` the optimizer keeps a 32-bit copy of all of them, updates that and rounds it to the tensors; without, a 16-bit tensor is
    updated in 32 bits and rounded each step. Arithmetic is 32-bit throughout.

    state_bits 8 holds the averages m and v in one byte each with a power of two for each 256 values (2.03 bytes a weight
    for both against 8), stochastically rounded from `seed`, the step and the position, so that runs repeat bit for bit: rounded to nearest,
    averages that move by 0.1% a step would stand still between values 6 to 12% apart. A gradient that is not
    finite turns its block of 256 to NaN.

    The state is flat: tensor i's starts at offsets[i], a multiple of 256. A tensor whose gradient is None is left alone, its
    step count with it.
    """

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2, state_bits: int = 32,
                 master: bool = False, seed: int = 0):
        self.params = list(params)
        if not self.params:
            raise ValueError("no parameters")
        for p in self.params:
            _on_gpu("a parameter", p, tuple(_CODE))
            if not p.is_contiguous() or p.device != self.params[0].device:
                raise ValueError("parameters are contiguous and on one device")
        spans = sorted((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size()) for p in self.params if p.numel())
        if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
            raise ValueError("parameters overlap")
        if state_bits not in (8, 32):
            raise ValueError(f"states are held in 8 or 32 bits, not {state_bits}")
        if lr < 0 or eps < 0 or weight_decay < 0 or not all(0 <= b < 1 for b in betas):
            raise ValueError("lr, eps and weight_decay must not be negative, betas in [0, 1)")
        self.lr, self.betas, self.eps, self.weight_decay = lr, tuple(betas), eps, weight_decay
        self.state_bits, self.seed, self.calls = state_bits, seed, 0
        self.device = self.params[0].device
        n = len(self.params)
        numel = np.array([p.numel() for p in self.params], np.int64)
        padded = -(-numel // STATE_BLOCK) * STATE_BLOCK
        self.offsets = np.concatenate([[0], np.cumsum(padded)])[:-1].tolist()
        self.size = int(padded.sum())
        chunks = -(-numel // CHUNK)
        self._first = np.concatenate([[0], np.cumsum(chunks)]).astype(np.int64)
        if self._first[-1] >= 2 ** 31:
            raise ValueError("too many weights")
        table = np.zeros(n, _TENSOR)
        table["param"], table["numel"], table["state_offset"] = [p.data_ptr() for p in self.params], numel, self.offsets
        table["param_type"], table["first_chunk"] = [_CODE[p.dtype] for p in self.params], self._first[:-1]
        self._table = torch.from_numpy(table.view(np.uint8).copy()).to(self.device)
        self._chunk_tensor = torch.from_numpy(np.repeat(np.arange(n, dtype=np.int32), chunks)).to(self.device)
        self._pointers = table["param"].tolist()
        self._shapes = [p.shape for p in self.params]
        self.steps = np.zeros(n, np.int32)
        kind = torch.uint8 if state_bits == 8 else torch.float32
        zeros = lambda k, t: torch.zeros(k, dtype=t, device=self.device)  # noqa: E731
        self.exp_avg, self.exp_avg_sq = zeros(self.size, kind), zeros(self.size, kind)
        self.exp_avg_exp, self.exp_avg_sq_exp = (zeros(self.size // STATE_BLOCK, torch.uint8) if state_bits == 8 else None for _ in range(2))
        self.master = zeros(self.size, torch.float32) if master else None
        if master:
            self.sync_master()

    def sync_master(self) -> None:
        """Takes the 32-bit copy from the tensors again, after something else has changed them."""
        for p, o in zip(self.params, self.offsets):
            self.master[o:o + p.numel()].copy_(p.detach().reshape(-1))

    def zero_grad(self) -> None:
        for p in self.params:
            p.grad = None

    def step(self, grads=None) -> None:
        """One step from `grads` (one tensor or None for each parameter, of its shape, any of the three types), or from the
        parameters' .grad. A gradient that is not contiguous is copied first."""
        grads = [p.grad for p in self.params] if grads is None else list(grads)
        if len(grads) != len(self.params):
            raise ValueError(f"{len(grads)} gradients for {len(self.params)} parameters")
        if [p.data_ptr() for p in self.params] != self._pointers:
            raise ValueError("a parameter has moved to other memory since the optimizer was made")
        types, steps = np.zeros(len(grads), np.int32), self.steps.copy()
        pointers = np.zeros(len(grads), np.uint64)
        for i, g in enumerate(grads):
            if g is None:
                continue
            if g.shape != self._shapes[i] or g.device != self.device or g.dtype not in _CODE:
                raise ValueError(f"gradient {i} must have its parameter's shape {tuple(self._shapes[i])}, be on its device, and be float32, bfloat16 or float16")
            if not g.is_contiguous():
                g = grads[i] = g.contiguous()
            pointers[i], types[i] = g.data_ptr(), _CODE[g.dtype]
            steps[i] += 1
        d = AdamwDesc()
        d.tensors, d.chunk_tensor, d.first_chunk = self._table.data_ptr(), self._chunk_tensor.data_ptr(), self._first.ctypes.data
        d.grads, d.grad_types, d.steps, d.n = pointers.ctypes.data, types.ctypes.data, steps.ctypes.data, len(grads)
        d.exp_avg, d.exp_avg_sq = self.exp_avg.data_ptr(), self.exp_avg_sq.data_ptr()
        if self.state_bits == 8:
            d.exp_avg_exp, d.exp_avg_sq_exp = self.exp_avg_exp.data_ptr(), self.exp_avg_sq_exp.data_ptr()
        d.master = None if self.master is None else self.master.data_ptr()
        d.lr, d.beta1, d.beta2, d.eps, d.weight_decay = self.lr, *self.betas, self.eps, self.weight_decay
        d.seed, d.calls, d.state_bits = self.seed, (self.calls + 1) & 0xffffffff, self.state_bits
        _call(self.device, library().ntc_op_adamw, C.byref(d))
        self.steps, self.calls = steps, self.calls + 1

    def moments(self):
        """m and v as 32-bit floats, flat (tensor i's at offsets[i]): the state itself, or with 8 bits the values it stands for."""
        if self.state_bits == 32:
            return self.exp_avg, self.exp_avg_sq
        m, v = (torch.empty(self.size, dtype=torch.float32, device=self.device) for _ in range(2))
        _call(self.device, library().ntc_op_adamw_moments, self.exp_avg.data_ptr(), self.exp_avg_sq.data_ptr(), self.exp_avg_exp.data_ptr(),
              self.exp_avg_sq_exp.data_ptr(), self.size, m.data_ptr(), v.data_ptr())
        return m, v

    def set_moments(self, m: torch.Tensor, v: torch.Tensor) -> None:
        """Takes m and v from 32-bit floats laid out as moments() gives them (to nearest, where the state has 8 bits)."""
        for t in (m, v):
            _on_gpu("a state", t, (torch.float32,))
            if t.numel() != self.size or not t.is_contiguous() or t.device != self.device:
                raise ValueError(f"a state has {self.size} contiguous values on the parameters' device")
        if self.state_bits == 32:
            self.exp_avg.copy_(m)
            self.exp_avg_sq.copy_(v)
        else:
            _call(self.device, library().ntc_op_adamw_encode, m.data_ptr(), v.data_ptr(), self.size, self.exp_avg.data_ptr(), self.exp_avg_sq.data_ptr(),
                  self.exp_avg_exp.data_ptr(), self.exp_avg_sq_exp.data_ptr())

    def state_dict(self) -> dict:
        return {"step": self.steps.tolist(), "calls": self.calls, "exp_avg": self.exp_avg, "exp_avg_sq": self.exp_avg_sq, "exp_avg_exp": self.exp_avg_exp,
                "exp_avg_sq_exp": self.exp_avg_sq_exp, "master": self.master}

    def load_state_dict(self, state: dict) -> None:
        """Copies a state_dict()'s contents. `step` may be one number for all tensors, `calls` is the largest step where it is absent,
        and the 32-bit copy is taken from the tensors where `master` is absent."""
        steps = np.broadcast_to(np.asarray(state["step"], np.int32), self.steps.shape)
        names = ["exp_avg", "exp_avg_sq"] + (["exp_avg_exp", "exp_avg_sq_exp"] if self.state_bits == 8 else [])
        for name in names + (["master"] if self.master is not None and state.get("master") is not None else []):
            mine, other = getattr(self, name), state.get(name)
            if other is None or other.shape != mine.shape or other.dtype != mine.dtype:
                raise ValueError(f"{name} must be {mine.dtype} of {mine.numel()} values")
            mine.copy_(other)
        if self.master is not None and state.get("master") is None:
            self.sync_master()
        self.steps = steps.copy()
        self.calls = int(state.get("calls", steps.max()))


# ---------------------------------------------------------------- 8-bit floating point in blocks
class Fp8Tensor(NamedTuple):
    """A matrix [R, K] in 8 bits: e4m3 codes (uint8 [R, K up to a multiple of 128], the rest 0) and exponent bytes E (scale 2^(E - 127);
    uint8 [blocks of rows, blocks of 128 columns up to a multiple of 4]) of blocks of `block_rows` (1 or 128) x 128."""
    codes: torch.Tensor
    exps: torch.Tensor
    shape: tuple
    block_rows: int

    def values(self) -> torch.Tensor:
        """The numbers it stands for, as 32-bit floats."""
        R, K = self.shape
        x = self.codes.view(torch.float8_e4m3fn).float()
        e = self.exps.to(torch.int32)
        scale = torch.where(e > 0, e << 23, 1 << 22).to(torch.int32).view(torch.float32)
        scale = scale.repeat_interleave(self.block_rows, 0)[:R].repeat_interleave(128, 1)[:, :x.shape[1]]
        return (x * scale)[:, :K]


def _fp8_empty(R: int, K: int, block_rows: int, device) -> Fp8Tensor:
    codes = torch.empty((R, -(-K // 128) * 128), dtype=torch.uint8, device=device)
    return Fp8Tensor(codes, torch.empty((-(-R // block_rows), -(-K // 512) * 4), dtype=torch.uint8, device=device), (R, K), block_rows)


def _quantize(x: torch.Tensor, block_rows: int, plain: bool, transposed: bool):
    _on_gpu("x", x, tuple(_CODE))
    if x.dim() != 2:
        raise ValueError(f"a matrix is needed, not {tuple(x.shape)}")
    if block_rows not in (1, 128):
        raise ValueError(f"blocks have 1 or 128 rows, not {block_rows}")
    x = x.detach()
    R, K = x.shape
    if (K > 1 and x.stride(1) != 1) or x.stride(0) < 0:
        x = x.contiguous()
    d = QuantizeDesc()
    d.x, d.R, d.K, d.row_stride, d.dtype, d.block_rows = x.data_ptr(), R, K, x.stride(0), _CODE[x.dtype], block_rows
    q = _fp8_empty(R, K, block_rows, x.device) if plain else None
    t = _fp8_empty(K, R, block_rows, x.device) if transposed else None
    if q is not None:
        d.codes, d.exps = q.codes.data_ptr(), q.exps.data_ptr()
    if t is not None:
        d.codes_t, d.exps_t = t.codes.data_ptr(), t.exps.data_ptr()
    if R and K:
        _call(x.device, library().ntc_op_fp8_quantize, C.byref(d))
    return q, t


def fp8_quantize(x: torch.Tensor, block_rows: int = 1) -> Fp8Tensor:
    """x [R, K] in 8 bits, a scale for each block_rows x 128 block: the smallest power of two that keeps the block within 448.
    Values are rounded to nearest (even); infinities become NaN."""
    return _quantize(x, block_rows, True, False)[0]


def fp8_quantize_t(x: torch.Tensor, block_rows: int = 1) -> Fp8Tensor:
    """x [R, K] transposed and in 8 bits, [K, R], its blocks along R: the operand of a product that sums over x's rows."""
    return _quantize(x, block_rows, False, True)[1]


def fp8_quantize_both(x: torch.Tensor, block_rows: int = 1):
    """(fp8_quantize(x), fp8_quantize_t(x)) from one read of x."""
    return _quantize(x, block_rows, True, True)


def _check_fp8(name: str, t) -> None:
    if not isinstance(t, Fp8Tensor):
        raise ValueError(f"{name} must be an Fp8Tensor")
    R, K = t.shape
    want = ((R, -(-K // 128) * 128), (-(-R // t.block_rows) if t.block_rows in (1, 128) else -1, -(-K // 512) * 4))
    for what, x, shape in zip(("codes", "exps"), (t.codes, t.exps), want):
        _on_gpu(f"{name}.{what}", x, (torch.uint8,))
        if tuple(x.shape) != shape or not x.is_contiguous() or x.device != t.codes.device or x.data_ptr() % 16:
            raise ValueError(f"{name}.{what} must be contiguous, start at a multiple of 16 bytes and be {shape} for a matrix {tuple(t.shape)} in blocks of {t.block_rows} x 128")


def _matmul(a, b: Fp8Tensor, dtype: torch.dtype) -> torch.Tensor:
    """a (an Fp8Tensor, or floats [M, K] that are taken to 8 bits on the way) times b transposed"""
    M, K = a.shape
    N, device = b.shape[0], b.codes.device
    c = torch.empty((M, N), dtype=dtype, device=device)
    if M == 0 or N == 0:
        return c
    if K == 0:
        return c.zero_()
    lib = library()
    size = lib.ntc_op_fp8_matmul_workspace(M, N, K)
    work = torch.empty(size, dtype=torch.uint8, device=device) if size else None
    d = MatmulDesc()
    if isinstance(a, Fp8Tensor):
        d.a, d.a_exps, d.a_type, d.a_block_rows = a.codes.data_ptr(), a.exps.data_ptr(), _FP8, a.block_rows
    else:
        d.a, d.a_stride, d.a_type, d.a_block_rows = a.data_ptr(), a.stride(0), _CODE[a.dtype], 1
    d.b, d.b_exps, d.b_block_rows = b.codes.data_ptr(), b.exps.data_ptr(), b.block_rows
    d.c, d.ldc, d.c_type, d.workspace = c.data_ptr(), N, _CODE[dtype], None if work is None else work.data_ptr()
    d.M, d.N, d.K = M, N, K
    _call(device, lib.ntc_op_fp8_matmul, C.byref(d))
    return c


def fp8_matmul(a: Fp8Tensor, b: Fp8Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """a [M, K] times b [N, K] transposed, summed in 32 bits and rounded once to dtype (bfloat16, float16 or float32; the 8-bit matrix
    instructions are good to 1.5e-5 of a result's magnitude, so float32 holds no more than that)."""
    _check_fp8("a", a)
    _check_fp8("b", b)
    if a.shape[1] != b.shape[1] or a.codes.device != b.codes.device:
        raise ValueError(f"a {tuple(a.shape)} and b {tuple(b.shape)} must have as many columns, on one device")
    if dtype not in _CODE:
        raise ValueError(f"products are float32, bfloat16 or float16, not {dtype}")
    return _matmul(a, b, dtype)


class _Fp8Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w):
        need_x, need_w = ctx.needs_input_grad
        xq, xt = _quantize(x, 1, True, need_w)
        wq, wt = _quantize(w, 128, True, need_x)
        ctx.kept = xt, wt, x.dtype, w.dtype
        return _matmul(xq, wq, x.dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        xt, wt, x_type, w_type = ctx.kept
        dq, dt = _quantize(dy, 1, wt is not None, xt is not None)
        return None if wt is None else _matmul(dq, wt, x_type), None if xt is None else _matmul(dt, xt, w_type)


def fp8_linear(x: torch.Tensor, w) -> torch.Tensor:
    """x [.., K] times w [N, K] transposed, in x's type, both taken to 8 bits (x in blocks of 1 x 128, w of 128 x 128).

    With w a tensor the layer is differentiable (once) in both: dx = q(dy) q(w) and dw = q(dy)^T q(x) with their
    operands in blocks along each product's own sum. With w an Fp8Tensor (fp8_quantize(w, 128), laid out once) it is for inference;
    few rows of x are then taken to 8 bits inside the product.
    """
    _on_gpu("x", x, tuple(_CODE))
    if x.dim() < 1:
        raise ValueError("x must have at least one axis")
    shape = x.shape
    if isinstance(w, Fp8Tensor):
        _check_fp8("w", w)
        if w.shape[1] != shape[-1] or w.codes.device != x.device:
            raise ValueError(f"x {tuple(shape)} must have w's {w.shape[1]} columns, on its device")
        if x.requires_grad and torch.is_grad_enabled():
            raise ValueError("w in 8 bits is for inference: give the weights themselves for a gradient")
        x = x.reshape(math.prod(shape[:-1]), shape[-1])
        if 0 < x.shape[0] <= library().ntc_op_fp8_matmul_float_rows() and shape[-1]:
            y = _matmul(x if x.stride(1) == 1 or shape[-1] == 1 else x.contiguous(), w, x.dtype)
        else:
            y = _matmul(fp8_quantize(x), w, x.dtype)
    else:
        _on_gpu("w", w, tuple(_CODE))
        if w.dim() != 2 or w.shape[1] != shape[-1] or w.device != x.device:
            raise ValueError(f"w {tuple(w.shape)} must be a matrix with x's {shape[-1]} columns, on its device")
        y = _Fp8Linear.apply(x.reshape(math.prod(shape[:-1]), shape[-1]), w)
    return y.view(*shape[:-1], y.shape[1])

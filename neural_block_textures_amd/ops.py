"""Operators of a learned prior over a texture's symbols, on torch tensors (the C ABI of include/ntc_ops.h).

    token_logprobs(logits, tokens, top=0)     log probabilities of given tokens, entropy, the best alternatives; differentiable
    AdamW(params, state_bits=32 or 8).step()  one step over many tensors
    fp8_quantize(x), fp8_matmul(a, b)         8-bit floating point with a power-of-two scale for each block of 128
    fp8_linear(x, w)                          a layer in it, for training or, with weights laid out once, for inference
    layer_norm(x, weight, bias)               rows to mean 0 and variance 1; differentiable, weight and bias too
    rotary(positions, q, k, sections=...)     rotary positions of several axes; differentiable
    attention(q, k, v, cu_q=..., cu_k=...)    causal attention over packed sequences or a cache, grouped heads; differentiable

Tensors are on the GPU; work is enqueued on torch's current stream and nothing waits. torch, or this module, has to be imported before
libntc_hip.so is loaded (by the first Trainer), so that both use one HIP runtime; the other order raises. Arguments that an operator does not
take (tensors with a forward-mode tangent among them) raise ValueError, errors of the runtime RuntimeError. There is no fallback: the kernels are libntc_hip.so's.
"""
from __future__ import annotations

import ctypes as C
import os
from typing import NamedTuple, Optional

import numpy as np
import torch

from . import trainer

STATE_BLOCK = 256
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


class LayerNormDesc(C.Structure):
    _fields_ = [("x", _P), ("weight", _P), ("bias", _P), ("y", _P), ("stats", _P), ("rows", _L), ("C", _L), ("x_stride", _L), ("dy_stride", _L), ("dtype", _I),
                ("weight_type", _I), ("eps", C.c_float), ("dy", _P), ("dx", _P), ("dweight", _P), ("dbias", _P), ("workspace", _P)]


class RotaryDesc(C.Structure):
    _fields_ = [("positions", _P), ("position_stride", _L), ("tokens", _L), ("x", _P * 2), ("y", _P * 2), ("token_stride", _L * 2), ("head_stride", _L * 2),
                ("heads", _I * 2), ("head_dim", _I), ("axes", _I), ("position_bytes", _I), ("dtype", _I), ("one_ladder", _I), ("interleaved", _I), ("backward", _I),
                ("sections", _I * 8), ("base", C.c_double)]


class AttentionDesc(C.Structure):
    _fields_ = [("q", _P), ("k", _P), ("v", _P), ("o", _P), ("o_rest", _P), ("lse", _P), ("cu_q", _P), ("cu_k", _P), ("k_lens", _P), ("sequences", _L), ("q_rows", _L), ("k_rows", _L),
                ("q_row_stride", _L), ("q_head_stride", _L), ("q_batch_stride", _L), ("k_row_stride", _L), ("k_head_stride", _L), ("k_batch_stride", _L),
                ("v_row_stride", _L), ("v_head_stride", _L), ("v_batch_stride", _L), ("q_heads", _I), ("k_heads", _I), ("head_dim", _I), ("dtype", _I), ("causal", _I),
                ("scale", C.c_float), ("workspace", _P), ("d_o", _P), ("do_row_stride", _L), ("do_head_stride", _L), ("do_batch_stride", _L), ("dq", _P), ("dk", _P),
                ("dv", _P)]


_TENSOR = np.dtype([("param", np.uint64), ("numel", np.int64), ("state_offset", np.int64), ("param_type", np.int32), ("first_chunk", np.int32)])
_lib = _bound = None


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
            "ntc_op_fp8_quantize_pair": (C.c_int, [_P, _P] + tail),
            "ntc_op_fp8_matmul_workspace": (C.c_size_t, [_L, _L, _L, _I]),
            "ntc_op_fp8_matmul": (C.c_int, [_P] + tail),
            "ntc_op_fp8_matmul_float_rows": (_L, []),
            "ntc_op_layer_norm": (C.c_int, [_P] + tail),
            "ntc_op_layer_norm_workspace": (C.c_size_t, [_L, _L]),
            "ntc_op_layer_norm_backward": (C.c_int, [_P] + tail),
            "ntc_op_rotary": (C.c_int, [_P] + tail),
            "ntc_op_attention_workspace": (C.c_size_t, [_P, _I]),
            "ntc_op_attention": (C.c_int, [_P] + tail),
            "ntc_op_attention_backward": (C.c_int, [_P] + tail),
        }
        for name, (res, args) in sig.items():
            fn = getattr(lib, name)
            fn.restype, fn.argtypes = res, args
        _lib = lib
    return _lib


def _binding():
    """The torch binding (_ops.so). Raises if it is not built: there is no other path."""
    global _bound
    if _bound is None:
        if not os.path.exists(os.path.join(trainer.PKG, "_ops.so")):
            raise RuntimeError("_ops.so is not built; run `python -m neural_block_textures_amd.build` (or __graft_entry__.build()) first")
        from . import _ops
        ours, torchs = _ops.runtimes()
        if ours != torchs:
            raise RuntimeError(f"two HIP runtimes are loaded, {ours} and torch's {torchs}, and a stream of one is none of the other: import torch (or "
                               "neural_block_textures_amd.ops) before the first use of neural_block_textures_amd.trainer")
        _bound = _ops
    return _bound


# ---------------------------------------------------------------- token log probabilities
class TokenLogprobs(NamedTuple):
    """What token_logprobs returns: in nats, 32-bit floats, in the tokens' shape (and one more axis for the alternatives)."""
    logprob: torch.Tensor
    entropy: torch.Tensor
    top_ids: Optional[torch.Tensor] = None
    top_logprobs: Optional[torch.Tensor] = None


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0, temperature: float = 1.0, ignore_index: int = -100) -> TokenLogprobs:
    """Log probabilities of `tokens` under softmax(logits / temperature), the distribution's entropy, and its `top` (at most 32)
    most probable symbols in descending order, equal ones by ascending index.

    logits [.., V]: float32, bfloat16 or float16, a row's values contiguous, rows at any two strides (a [batch, time, V] tensor's
    [:, :-1] as it lies). tokens [..]: int32 or int64. temperature: 2^-127 to 2^120. A token equal to ignore_index has logprob 0 and no gradient;
    another one outside [0, V) has logprob NaN. -inf masks a symbol; a row with nothing left has log probabilities -inf, entropy 0
    and gradient 0; a NaN or +inf makes its row's results NaN (ids then order NaN as -inf). logprob, entropy and top_logprobs are
    differentiable in logits (once); log probabilities and sums are 32-bit, dlogits is rounded once to the logits' type.
    """
    return TokenLogprobs(*_binding().token_logprobs(logits, tokens, top, temperature, ignore_index))


# ---------------------------------------------------------------- AdamW
class AdamW:
    """AdamW over many tensors in few launches, its state in 32 bits or in 8.

    params: contiguous GPU tensors (float32, bfloat16, float16, mixed as they come) of one device; they are updated in place. With
    `master` the optimizer keeps a 32-bit copy of all of them, updates that and rounds it to the tensors; without, a 16-bit tensor is
    updated in 32 bits and rounded each step. Arithmetic is 32-bit throughout.

    state_bits 8 holds the averages m and v in one byte each with a power of two for each 256 values (2.03 bytes a weight
    for both against 8), stochastically rounded from `seed`, the step and the position, so that runs repeat bit for bit: rounded to nearest,
    averages that move by 0.1% a step would stand still between values 6 to 12% apart. A gradient that is not
    finite turns its block of 256 to NaN. With eps 0 a weight whose gradients have all been 0 becomes NaN, as the formula's 0 / 0 is.

    The state is flat: tensor i's starts at offsets[i], a multiple of 256. A tensor whose gradient is None is left alone, its
    step count with it.
    """

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2, state_bits: int = 32,
                 master: bool = False, seed: int = 0):
        self.params = list(params)
        if not self.params:
            raise ValueError("no parameters")
        if state_bits not in (8, 32):
            raise ValueError(f"states are held in 8 or 32 bits, not {state_bits}")
        if not (lr >= 0 and eps >= 0 and weight_decay >= 0) or len(betas) != 2 or not all(0 <= b < 1 for b in betas):
            raise ValueError("lr, eps and weight_decay must not be negative, the two betas in [0, 1)")
        if not 0 <= seed < 2 ** 64:
            raise ValueError(f"seed must be from 0 to 2^64 - 1, not {seed}")
        self._plan = _binding().AdamwPlan(self.params)
        self.lr, self.betas, self.eps, self.weight_decay = lr, tuple(betas), eps, weight_decay
        self.state_bits, self.seed = state_bits, seed
        self.device, self.offsets, self.size = self.params[0].device, self._plan.offsets, self._plan.size
        kind = torch.uint8 if state_bits == 8 else torch.float32
        zeros = lambda k, t: torch.zeros(k, dtype=t, device=self.device)  # noqa: E731
        self.exp_avg, self.exp_avg_sq = zeros(self.size, kind), zeros(self.size, kind)
        self.exp_avg_exp, self.exp_avg_sq_exp = (zeros(self.size // STATE_BLOCK, torch.uint8) if state_bits == 8 else None for _ in range(2))
        self.master = zeros(self.size, torch.float32) if master else None
        if master:
            self.sync_master()

    @property
    def steps(self) -> np.ndarray:
        """How many steps each tensor has taken."""
        return np.array(self._plan.steps, np.int32)

    @property
    def calls(self) -> int:
        return self._plan.calls

    def sync_master(self) -> None:
        """Takes the 32-bit copy from the tensors again, after something else has changed them."""
        for p, o in zip(self.params, self.offsets):
            self.master[o:o + p.numel()].copy_(p.detach().reshape(-1))

    def zero_grad(self) -> None:
        for p in self.params:
            p.grad = None

    def step(self, grads=None) -> None:
        """One step from `grads` (one tensor or None for each parameter, of its shape, any of the three types), or from the
        parameters' .grad. A gradient that is not contiguous is copied first. In a captured graph a replay is this same step again: the same
        step count, rates and random bits, and not counted."""
        self._plan.step(grads, self.exp_avg, self.exp_avg_sq, self.exp_avg_exp, self.exp_avg_sq_exp, self.master, self.state_bits, self.lr, *self.betas,
                        self.eps, self.weight_decay, self.seed)

    def moments(self):
        """m and v as 32-bit floats, flat (tensor i's at offsets[i]): the state itself, or with 8 bits the values it stands for."""
        if self.state_bits == 32:
            return self.exp_avg, self.exp_avg_sq
        return _binding().adamw_moments(self.exp_avg, self.exp_avg_sq, self.exp_avg_exp, self.exp_avg_sq_exp)

    def set_moments(self, m: torch.Tensor, v: torch.Tensor) -> None:
        """Takes m and v from 32-bit floats laid out as moments() gives them (to nearest, where the state has 8 bits)."""
        for t in (m, v):
            if t.dtype != torch.float32 or t.numel() != self.size or not t.is_contiguous() or t.device != self.device:
                raise ValueError(f"a state has {self.size} contiguous 32-bit values on the parameters' device")
        if self.state_bits == 32:
            self.exp_avg.copy_(m)
            self.exp_avg_sq.copy_(v)
        else:
            _binding().adamw_encode(m, v, self.exp_avg, self.exp_avg_sq, self.exp_avg_exp, self.exp_avg_sq_exp)

    def state_dict(self) -> dict:
        return {"step": list(self._plan.steps), "calls": self.calls, "exp_avg": self.exp_avg, "exp_avg_sq": self.exp_avg_sq, "exp_avg_exp": self.exp_avg_exp,
                "exp_avg_sq_exp": self.exp_avg_sq_exp, "master": self.master, "seed": self.seed}

    def load_state_dict(self, state: dict) -> None:
        """Copies a state_dict()'s contents; one that does not fit changes nothing. `step` may be one number for all tensors, `calls` is the
        largest step where it is absent, the 32-bit copy is taken from the tensors where `master` is absent, and the optimizer's own seed
        stays where `seed` is absent (a run goes on bit for bit on its first one's)."""
        steps = np.asarray(state["step"])
        if steps.shape not in ((), (1,), (len(self.params),)) or not ((steps >= 0) & (steps < 2 ** 31 - 1) & (steps == np.floor(steps))).all():
            raise ValueError(f"step must be one count from 0 on, or {len(self.params)}")
        steps = np.broadcast_to(steps, (len(self.params),)).astype(np.int32).tolist()
        calls = int(state.get("calls", max(steps)))
        if calls < 0:
            raise ValueError(f"calls must be a count from 0 on, not {calls}")
        seed = int(state.get("seed", self.seed))
        if not 0 <= seed < 2 ** 64:
            raise ValueError(f"seed must be from 0 to 2^64 - 1, not {seed}")
        names = ["exp_avg", "exp_avg_sq"] + (["exp_avg_exp", "exp_avg_sq_exp"] if self.state_bits == 8 else [])
        names += ["master"] if self.master is not None and state.get("master") is not None else []
        for name in names:
            mine, other = getattr(self, name), state.get(name)
            if other is None or other.shape != mine.shape or other.dtype != mine.dtype:
                raise ValueError(f"{name} must be {mine.dtype} of {mine.numel()} values")
        for name in names:
            getattr(self, name).copy_(state[name])
        if self.master is not None and state.get("master") is None:
            self.sync_master()
        self._plan.steps = steps
        self._plan.calls = calls
        self.seed = seed


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


def _quantize(x: torch.Tensor, block_rows: int, plain: bool, transposed: bool):
    q, t = _binding().quantize(x, block_rows, plain, transposed)
    R, K = x.shape
    return q and Fp8Tensor(*q, (R, K), block_rows), t and Fp8Tensor(*t, (K, R), block_rows)


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


def fp8_matmul(a: Fp8Tensor, b: Fp8Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """a [M, K] times b [N, K] transposed, summed in 32 bits and rounded once to dtype (bfloat16, float16 or float32). K is at most
    2^23. The 8-bit matrix instruction cuts each product off 13 bits below the largest of its eight neighbours: 1.5e-5 of a result's magnitude on random
    values, more in rows that lie far below their block's largest (subnormal codes), so that float32 holds no more than that."""
    for name, t in (("a", a), ("b", b)):
        if not isinstance(t, Fp8Tensor):
            raise ValueError(f"{name} must be an Fp8Tensor")
    return _binding().matmul(a.codes, a.exps, *a.shape, a.block_rows, b.codes, b.exps, *b.shape, b.block_rows, dtype)


def fp8_linear(x: torch.Tensor, w) -> torch.Tensor:
    """x [.., K] times w [N, K] transposed, in x's type, both taken to 8 bits (x in blocks of 1 x 128, w of 128 x 128).

    With w a tensor the layer is differentiable (once) in both: dx = q(dy) q(w) and dw = q(dy)^T q(x) with their
    operands in blocks along each product's own sum. With w an Fp8Tensor (fp8_quantize(w, 128), laid out once) it is for inference;
    few rows of x are then taken to 8 bits inside the product. Sums are fp8_matmul's, good to about 1.5e-5 of a result's magnitude: a 32-bit y holds no
    more than that. K is at most 2^23 (and N, for a gradient in x); rows may be any number.
    """
    if isinstance(w, Fp8Tensor):
        return _binding().linear_fp8(x, w.codes, w.exps, *w.shape, w.block_rows)
    return _binding().linear(x, w)


# ---------------------------------------------------------------- the blocks of a sequence model
def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(variance + eps) * weight + bias over x's last axis, in x's type.

    x [.., C]: float32, bfloat16 or float16 (copied first where a row's values are not contiguous or rows lie at several strides). weight and bias [C]:
    of x's type or float32, both alike, or None. Differentiable (once) in all three. Statistics and sums are 32-bit, the weight's and bias's gradients over the rows too,
    in an order that depends on the sizes alone; a row with a value that is not finite is NaN.
    """
    return _binding().layer_norm(x, weight, bias, eps)


def rotary(positions: torch.Tensor, q: torch.Tensor, k: Optional[torch.Tensor] = None, *, sections, base: float = 10000.0, one_ladder: bool = False,
           interleaved: bool = False):
    """q, or (q, k), with pairs of each head's elements turned by angles that grow with the token's positions.

    positions [.., axes]: int32 or int64, a token's place on each of 1 to 8 axes (time, row, column, channel). q and k [.., heads, elements]: float32, bfloat16 or float16, any
    strides. sections: how many pairs of a head each axis turns, 128 in all at most; pair p of P is elements p and p + P, or with `interleaved` 2p and 2p + 1, and elements from 2 P on
    stay as they are. Axis a's pair j turns by its position times base^(-j / sections[a]); with one_ladder pair p by its axis's position times base^(-p / P).
    Angles are made in 64 bits, and off by no more than the position times (2^-57 of the frequency + 2^-65 of a turn): 2^-24 at 2^33. Sines, cosines and sums are 32-bit, rounded once.
    Differentiable (once) in q and k.
    """
    out = _binding().rotary(positions, q, k, list(sections), base, one_ladder, interleaved)
    return out[0] if k is None else out


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, causal: bool = True, scale: Optional[float] = None, cu_q: Optional[torch.Tensor] = None,
              cu_k: Optional[torch.Tensor] = None, k_lens: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(scale q k^T) v for each sequence and head, in q's type and shape. With `causal` query i of a sequence of Lq queries and Lk keys sees keys up to
    i + Lk - Lq: the last query sees all of them. A query that sees none has 0, and no gradient.

    q [sequences, rows, heads, elements], or packed [rows, heads, elements] with cu_q (int32 [sequences + 1] on the GPU: 0 and each sequence's end, ascending; without it one
    sequence). k and v alike, with cu_k; their heads divide q's, and query head h reads key head h // (q's heads / k's). k_lens (int32 [sequences]): how many of its
    rows of k and v a sequence has, as with a cache that has room; the rest are not read. Rows behind the last end have 0. scale: 1 / sqrt(elements) where it is None.

    bfloat16 or float16, 8 to 128 elements a head (a multiple of 8), any strides (copied first where heads are not contiguous, or not at multiples of 16 bytes). Differentiable (once) in
    q, k and v. Scores, the softmax and sums are 32-bit; probabilities, and backwards the scores' gradients, are rounded to the tensors' type for the products that
    follow. Nothing is added by atomics: results repeat bit for bit. Lengths are read on the GPU: numbers that leave the tensors are cut off there, and give wrong results, not an error. A key or
    value that is not finite makes the queries that see it NaN where the formula does, and possibly any other of its sequence; a query whose scores are all -inf is NaN.
    """
    return _binding().attention(q, k, v, causal, scale, cu_q, cu_k, k_lens)

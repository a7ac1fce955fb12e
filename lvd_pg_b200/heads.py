"""What stands between a network's categorical head and a circuit (include/pcb200.h, "categorical heads"):

  token_logprobs   log-probabilities of given categories, entropy and best alternatives of logits, differentiable
  soft_evidence    logits [rows, vars, cats] as the soft evidence that `forward_ex`, `em_step_ex` and
                   `mini_batch_em_soft` take, differentiable
  QuantHead        a head whose weights are held in 4 bits with group scales, for few feature vectors at a time

The reference trains its teachers in PyTorch (src/models/, src/maskedAE, src/pixelcnn) and hands their outputs to the
circuits as arrays; these run on the GPU beside the circuit.  Every call is enqueued on the current stream of its tensors'
device, allocates through torch's allocator alone and does not synchronise.  Forward and backward passes can be captured into
CUDA graphs; as for every torch operator, a captured backward pass needs leaves of its own (made in the capture, as
`static.detach().requires_grad_()`): with leaves that an eager graph still holds, torch waits for that graph's stream and the
capture fails.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad

from . import _lib

MAX_ALTERNATIVES = 32
MOST = 2 ** 31 - 1   # categories, variables, features that the library is told of in 32 bits
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


class TokenLogprobs(NamedTuple):
    logp: Optional[torch.Tensor]       # float32, the shape of the tokens; None without tokens
    entropy: torch.Tensor              # float32
    top_ids: Optional[torch.Tensor]    # int64 [..., top_k], best first; None without alternatives
    top_logp: Optional[torch.Tensor]   # float32


def _need(ok: bool, message: str) -> None:
    if not ok:
        raise _lib.PcbError(1, message)


def _call(dev: torch.device, fn, *args) -> None:
    """`fn` on the current stream of `dev`, which becomes the current device for the call where it is not."""
    if torch.cuda.current_device() == dev.index:
        code = fn(*args, torch._C._cuda_getCurrentRawStream(dev.index))
    else:
        with torch.cuda.device(dev):
            code = fn(*args, torch._C._cuda_getCurrentRawStream(dev.index))
    if code != 0:
        _lib.check(code)


def _no_tangent(x: torch.Tensor) -> None:
    """These operators are differentiated backwards; a tangent of forward mode would be lost without a word."""
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(x).tangent is not None:   # (the level first: a microsecond less)
        _need(False, "no forward-mode derivatives: the argument carries a tangent")


def _logits(x: torch.Tensor) -> int:
    if not (isinstance(x, torch.Tensor) and x.is_cuda):
        _need(False, "logits must be a CUDA tensor; there is no CPU fallback")
    dtype = _DTYPES.get(x.dtype)
    if dtype is None:
        _need(False, "logits are float32, bfloat16 or float16")
    if x.dim() < 1 or x.shape[-1] < 1:
        _need(False, "logits need at least one category")
    if x.shape[-1] > MOST:
        _need(False, "logits have at most 2^31 - 1 categories")
    _no_tangent(x)
    return dtype


def _once() -> None:
    """Called in a backward pass: gradients are enabled there only where a gradient of the gradient is asked for."""
    if torch.is_grad_enabled():
        raise RuntimeError("pcb200: this operator can be differentiated once only (create_graph=True is not supported)")


# ---- log-probabilities --------------------------------------------------------------------------------------
def _logprobs_forward(x2, tokens, top_k, temperature, dtype, stats=None):
    rows, cats = x2.shape
    dev = x2.device
    entropy = torch.empty(rows, dtype=torch.float32, device=dev)
    logp = None if tokens is None else torch.empty(rows, dtype=torch.float32, device=dev)
    top_ids = torch.empty((rows, top_k), dtype=torch.int64, device=dev) if top_k else None
    top_logp = torch.empty((rows, top_k), dtype=torch.float32, device=dev) if top_k else None
    _call(dev, _lib.lib().pcb_token_logprobs, x2.data_ptr(), dtype, rows, cats, x2.stride(0), temperature,
          None if tokens is None else tokens.data_ptr(), 0 if tokens is None else tokens.element_size(), top_k,
          None if tokens is None else logp.data_ptr(), entropy.data_ptr(), None if stats is None else stats.data_ptr(),
          top_ids.data_ptr() if top_k else None, top_logp.data_ptr() if top_k else None)
    return logp, entropy, top_ids, top_logp


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x2, tokens, top_k, temperature, dtype):
        stats = torch.empty((x2.shape[0], 2), dtype=torch.float32, device=x2.device)
        logp, entropy, top_ids, top_logp = _logprobs_forward(x2, tokens, top_k, temperature, dtype, stats)
        ctx.save_for_backward(x2, tokens, stats, entropy, top_ids)
        ctx.top_k, ctx.temperature, ctx.dtype = top_k, temperature, dtype
        ctx.set_materialize_grads(False)
        if top_ids is not None:
            ctx.mark_non_differentiable(top_ids)
        return logp, entropy, top_ids, top_logp

    @staticmethod
    def backward(ctx, g_logp, g_entropy, _, g_top):
        _once()
        x2, tokens, stats, entropy, top_ids = ctx.saved_tensors
        if g_logp is None and g_entropy is None and g_top is None:
            return None, None, None, None, None
        rows, cats = x2.shape
        dx = torch.empty(rows, cats, dtype=x2.dtype, device=x2.device)
        g_top = None if g_top is None else g_top.contiguous()
        _call(x2.device, _lib.lib().pcb_token_logprobs_backward, x2.data_ptr(), ctx.dtype, rows, cats, x2.stride(0), ctx.temperature,
              None if tokens is None else tokens.data_ptr(), 0 if tokens is None else tokens.element_size(), ctx.top_k,
              None if top_ids is None else top_ids.data_ptr(), stats.data_ptr(), entropy.data_ptr(),
              None if g_logp is None else g_logp.data_ptr(), 0 if g_logp is None else g_logp.stride(0),
              None if g_entropy is None else g_entropy.data_ptr(), 0 if g_entropy is None else g_entropy.stride(0),
              None if g_top is None else g_top.data_ptr(), dx.data_ptr())
        return dx, None, None, None, None


def token_logprobs(logits: torch.Tensor, tokens: Optional[torch.Tensor] = None, top_k: int = 0,
                   temperature: float = 1.0) -> TokenLogprobs:
    """Scores of `logits` [..., cats] (float32, bfloat16 or float16; any strides), with logp = log_softmax(logits / temperature):
    the log-probability of `tokens` [...] (int32 or int64), the entropy, and the `top_k` <= 32 best alternatives with their
    log-probabilities, of equal logits the lowest index first.  Everything is float32 and differentiable with respect to
    the logits (not twice, and backwards only: a tangent of forward mode is refused).

    A negative token means that none is given: its log-probability is 0, its gradient nothing.  One past the last category
    gives NaN.  A row of -inf throughout has log-probabilities -inf, entropy 0 and gradient 0; a row with NaN or +inf is NaN."""
    dtype = _logits(logits)
    cats = logits.shape[-1]
    _need(0 <= top_k <= MAX_ALTERNATIVES and top_k <= cats, "top_k must be between 0 and 32, and no more than there are categories")
    _need(0.0 < temperature < float("inf"), "the temperature must be positive and finite")
    shape = logits.shape[:-1]
    x2 = logits if logits.dim() == 2 else logits.reshape(-1, cats)
    if x2.stride(1) != 1 and cats > 1:
        x2 = x2.contiguous()
    if tokens is not None:
        _need(isinstance(tokens, torch.Tensor) and tokens.device == logits.device and tokens.dtype in (torch.int64, torch.int32),
              "tokens must be int32 or int64 on the logits' device")
        _need(tokens.shape == shape, "tokens must have the logits' shape without the last axis")
        tokens = tokens.contiguous()
    if torch.is_grad_enabled() and logits.requires_grad:
        logp, entropy, top_ids, top_logp = _TokenLogprobs.apply(x2, tokens, top_k, temperature, dtype)
    else:
        logp, entropy, top_ids, top_logp = _logprobs_forward(x2, tokens, top_k, temperature, dtype)
    if logits.dim() != 2:
        entropy = entropy.view(shape)
        if tokens is not None:
            logp = logp.view(shape)
        if top_k:
            top_ids, top_logp = top_ids.view(shape + (top_k,)), top_logp.view(shape + (top_k,))
    return TokenLogprobs(logp, entropy, top_ids, top_logp)


# ---- soft evidence ------------------------------------------------------------------------------------------
def _evidence_forward(x, miss, temperature, dtype, stats):
    rows, variables, cats = x.shape
    out = torch.empty_strided(x.shape, (1, rows, rows * variables), dtype=torch.float32, device=x.device)
    _call(x.device, _lib.lib().pcb_soft_evidence, x.data_ptr(), dtype, rows, variables, cats, x.stride(0), x.stride(1),
          None if miss is None else miss.data_ptr(), 0 if miss is None else miss.stride(0), 0 if miss is None else miss.stride(1),
          temperature, out.data_ptr(), None if stats is None else stats.data_ptr())
    return out


class _SoftEvidence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, miss, temperature, dtype):
        stats = torch.empty((x.shape[0], x.shape[1], 2), dtype=torch.float32, device=x.device)
        out = _evidence_forward(x, miss, temperature, dtype, stats)
        ctx.save_for_backward(x, miss, stats)
        ctx.temperature, ctx.dtype = temperature, dtype
        return out

    @staticmethod
    def backward(ctx, g):
        _once()
        x, miss, stats = ctx.saved_tensors
        rows, variables, cats = x.shape
        if g.stride() != (1, rows, rows * variables):   # not laid out as the evidence is
            g = g.permute(2, 1, 0).contiguous()
        dx = torch.empty((rows, variables, cats), dtype=x.dtype, device=x.device)
        _call(x.device, _lib.lib().pcb_soft_evidence_backward, x.data_ptr(), ctx.dtype, rows, variables, cats, x.stride(0), x.stride(1),
              None if miss is None else miss.data_ptr(), 0 if miss is None else miss.stride(0), 0 if miss is None else miss.stride(1),
              ctx.temperature, stats.data_ptr(), g.data_ptr(), dx.data_ptr())
        return dx, None, None, None


def soft_evidence(logits: torch.Tensor, miss: Optional[torch.Tensor] = None, temperature: float = 1.0) -> torch.Tensor:
    """A network's `logits` [rows, vars, cats] (float32, bfloat16 or float16; any strides) as soft evidence: float32
    log-weights log_softmax(logits / temperature) [rows, vars, cats] with the row index fastest, as `forward_ex(soft=...)`,
    `em_step_ex` and `mini_batch_em_soft` take them (regularization/reg_likelihood.jl:51-91).  A variable that is missing in
    a row (`miss` [rows, vars], bool or uint8) weighs all its categories alike: 0.  Differentiable with respect to the logits
    (not twice, and not in forward mode); where missing, or where all logits are -inf (evidence -inf throughout), the gradient
    is 0."""
    dtype = _logits(logits)
    _need(logits.dim() == 3, "logits must be [rows, vars, cats]")
    _need(logits.shape[1] <= MOST, "soft evidence has at most 2^31 - 1 variables")
    _need(0.0 < temperature < float("inf"), "the temperature must be positive and finite")
    if miss is not None:
        _need(isinstance(miss, torch.Tensor) and miss.device == logits.device and miss.dtype in (torch.bool, torch.uint8),
              "miss must be bool or uint8 on the logits' device")
        _need(miss.shape == logits.shape[:2], "miss must be [rows, vars]")
    x = logits if logits.stride(2) == 1 or logits.shape[2] == 1 else logits.contiguous()
    if torch.is_grad_enabled() and logits.requires_grad:
        return _SoftEvidence.apply(x, miss, temperature, dtype)
    return _evidence_forward(x, miss, temperature, dtype, None)


# ---- a head in 4 bits ---------------------------------------------------------------------------------------
class QuantHead:
    """A categorical head y = x W^T + bias for serving, its weights W [cats, features] in 4 bits: W[n, k] =
    scales[n, k // group] * (code - 8), codes 0..15, 16-bit scales.  `QuantHead(weight)` quantises (scale = max |w| / 7 of the
    group, which NaN or an infinite weight makes NaN throughout); `QuantHead.from_codes` takes codes and scales that another
    program made.  The weights are laid out once, on construction, on the weight's device; calls keep nothing.  A captured
    graph holds their address: keep the head while it lives.  For inference: features that require a gradient or carry a
    tangent are refused."""

    def __init__(self, weight: torch.Tensor, group: int = 64, bias: Optional[torch.Tensor] = None):
        _need(isinstance(weight, torch.Tensor) and weight.is_cuda and weight.dim() == 2 and weight.dtype in _DTYPES,
              "weight must be a [cats, features] CUDA tensor of float32, bfloat16 or float16")
        _need(1 <= weight.shape[0] <= MOST and 1 <= weight.shape[1] <= MOST, "a head has 1 to 2^31 - 1 categories and at least one feature")
        _need(group in (32, 64, 128), "groups hold 32, 64 or 128 features")
        w = weight.detach().contiguous()
        cats, features = w.shape
        codes = torch.empty((cats, (features + 1) // 2), dtype=torch.uint8, device=w.device)
        scales = torch.empty((cats, -(-features // group)), device=w.device,
                             dtype=torch.float16 if w.dtype == torch.float16 else torch.bfloat16)
        _call(w.device, _lib.lib().pcb_head_quantize, w.data_ptr(), _DTYPES[w.dtype], cats, features, group, _DTYPES[scales.dtype],
              codes.data_ptr(), scales.data_ptr())
        self._pack(codes, scales, features, group, bias)

    @classmethod
    def from_codes(cls, codes: torch.Tensor, scales: torch.Tensor, features: int, group: int = 64,
                   bias: Optional[torch.Tensor] = None) -> "QuantHead":
        """codes [cats, ceil(features / 2)] uint8, two a byte, the even feature in the low half; scales
        [cats, ceil(features / group)] bfloat16 or float16."""
        _need(group in (32, 64, 128), "groups hold 32, 64 or 128 features")
        _need(isinstance(codes, torch.Tensor) and codes.is_cuda and codes.dtype == torch.uint8 and codes.dim() == 2,
              "codes must be a uint8 CUDA matrix")
        cats = codes.shape[0]
        _need(1 <= cats <= MOST and 1 <= features <= MOST and codes.shape[1] == (features + 1) // 2, "codes must be [cats, ceil(features / 2)]")
        _need(isinstance(scales, torch.Tensor) and scales.device == codes.device and scales.dtype in (torch.bfloat16, torch.float16),
              "scales must be bfloat16 or float16 on the codes' device")
        _need(tuple(scales.shape) == (cats, -(-features // group)), "scales must be [cats, ceil(features / group)]")
        self = cls.__new__(cls)
        self._pack(codes.contiguous(), scales.contiguous(), features, group, bias)
        return self

    def _pack(self, codes, scales, features, group, bias):
        self.cats, self.features, self.group, self.device = int(codes.shape[0]), int(features), int(group), codes.device
        if bias is not None:
            _need(isinstance(bias, torch.Tensor) and bias.device == self.device and tuple(bias.shape) == (self.cats,),
                  "bias must be [cats] on the codes' device")
            bias = bias.detach().to(torch.float32, copy=True).contiguous()
        self.bias, self._scale_dtype = bias, _DTYPES[scales.dtype]
        lib, size = _lib.lib(), C.c_uint64()
        _lib.check(lib.pcb_head_packed_bytes(self.cats, self.features, self.group, C.byref(size)))
        self.packed = torch.empty(size.value, dtype=torch.uint8, device=self.device)
        _call(self.device, lib.pcb_head_pack, codes.data_ptr(), scales.data_ptr(), self.cats, self.features, self.group,
              self.packed.data_ptr())
        self._made_on = torch._C._cuda_getCurrentRawStream(self.device.index)

    def _hold(self) -> None:
        """Weights that another stream than their own reads are not handed out again before it is done."""
        if torch._C._cuda_getCurrentRawStream(self.device.index) != self._made_on:
            stream = torch.cuda.current_stream(self.device)
            self.packed.record_stream(stream)
            if self.bias is not None:
                self.bias.record_stream(stream)

    def weight(self) -> torch.Tensor:
        """The weights that the codes stand for, [cats, features] float32."""
        self._hold()
        out = torch.empty((self.cats, self.features), dtype=torch.float32, device=self.device)
        _call(self.device, _lib.lib().pcb_head_weight, self.packed.data_ptr(), self._scale_dtype, self.cats, self.features, self.group,
              out.data_ptr())
        return out

    def logits(self, x: torch.Tensor, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        """x [..., features] (float32, bfloat16 or float16) -> [..., cats] in `out_dtype` (default: x's type).  Sums are
        float32, a group's before its scale: features up to 3.3e35 in magnitude keep them in range.  Meant for few rows: up
        to 32 of them (10 of float32; fewer beyond about 2400 features, 21 and 7 at 4096) read the weights once."""
        _need(isinstance(x, torch.Tensor) and x.device == self.device and x.dtype in _DTYPES,
              "features must be float32, bfloat16 or float16 on the head's device")
        if x.dim() < 1 or x.shape[-1] != self.features:
            _need(False, f"features must end in {self.features} values")
        _need(not (x.requires_grad and torch.is_grad_enabled()), "a head in 4 bits gives no gradient: detach the features")
        _no_tangent(x)
        out_dtype = out_dtype or x.dtype
        _need(out_dtype in _DTYPES, "logits are float32, bfloat16 or float16")
        x2 = x if x.dim() == 2 else x.reshape(-1, self.features)
        if x2.stride(1) != 1 and self.features > 1:
            x2 = x2.contiguous()
        self._hold()
        y = torch.empty((x2.shape[0], self.cats), dtype=out_dtype, device=self.device)
        _call(self.device, _lib.lib().pcb_head_logits, self.packed.data_ptr(), self._scale_dtype, self.cats, self.features, self.group,
              x2.data_ptr(), _DTYPES[x.dtype], x2.shape[0], x2.stride(0), None if self.bias is None else self.bias.data_ptr(), y.data_ptr(),
              _DTYPES[out_dtype])
        return y if x.dim() == 2 else y.view(x.shape[:-1] + (self.cats,))

    def logprobs(self, x: torch.Tensor, tokens: Optional[torch.Tensor] = None, top_k: int = 0, temperature: float = 1.0) -> TokenLogprobs:
        """`token_logprobs` of this head's float32 logits."""
        return token_logprobs(self.logits(x, torch.float32), tokens, top_k, temperature)

    def evidence(self, x: torch.Tensor, miss: Optional[torch.Tensor] = None, temperature: float = 1.0) -> torch.Tensor:
        """`soft_evidence` of this head's float32 logits for features [rows, vars, features]: one head for every variable."""
        _need(isinstance(x, torch.Tensor) and x.dim() == 3, "features must be [rows, vars, features]")
        return soft_evidence(self.logits(x, torch.float32), miss, temperature)

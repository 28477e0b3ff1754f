"""A mixture-of-experts layer around the NVFP4 products, with the group sizes on the device.

The grouped GEMM (eval/nvfp4_grouped_gemm/reference.py:137-201) takes its group sizes as a host list.  Here the router
runs on the GPU and nothing is copied back: every call is asynchronous on the current stream and can be captured into
a graph.  One layer:

    r = moe.route(logits, top_k)                                     # weights, experts, plan
    a, sfa = moe.dispatch_nvfp4(x, r.plan)                           # tokens sorted by expert, quantised
    h, sfh = moe.expert_dual_gemm_nvfp4(a, sfa, b1, sfb1, b2, sfb2, r.plan)
    y = moe.expert_gemm(h, sfh, b3, sfb3, r.plan)                    # fp16 rows, sorted by expert
    out = moe.combine(y, r.plan, r.weights, dtype=x.dtype)

T tokens choose k of E experts each.  Copy ``i = t * k + j`` is choice j of token t; the copies are sorted stably by
expert into ``T * k`` rows.  A choice whose expert id lies outside [0, E) (-1, say) is not routed and has no row; the rows
behind the last routed copy are zero in every sorted buffer made here.

Expert weights are one batched operand, as ``quantize.quantize_operand`` makes it of ``[E, N, K]``: packed codes
``[N, K/2, E]`` and the 6-D swizzled view of their scales.  The gradients of the 16- and 32-bit operations are functions
of their own (``*_backward``); there are none of the NVFP4 products.  Nothing here registers with autograd: results never
require gradients, whatever their inputs do, so a training step calls these functions from ``torch.autograd.Function``s
of its own.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _args, _lib

MAX_EXPERTS, MAX_CHOICES = 1024, 32
MAX_COPIES = (1 << 31) - (1 << 20)      # also of a matrix: rows, columns
_KINDS = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


class Plan:
    """How the copies of a batch are sorted (``nvfp4_moe_plan``).  One int32 buffer on the batch's device holds its six
    tables; the views are made when they are asked for (a call of the layer needs only their addresses)."""
    __slots__ = ("buffer", "num_tokens", "top_k", "num_experts", "num_copies", "most_tiles", "_at", "_more")

    def __init__(self, num_tokens: int, top_k: int, num_experts: int, device: torch.device, more: int = 0):
        n, e = num_tokens * top_k, num_experts + 1
        if n > MAX_COPIES:
            raise ValueError(f"expected at most {MAX_COPIES} choices in a batch, got {n}")
        # behind the tables: the copies per expert of each block of a large sort, then `more` words for the caller
        scratch = _lib.load().nvfp4_moe_plan_scratch(num_tokens, num_experts, top_k) // 4 if n > 4096 else 0
        self._more = 3 * e + 3 * n + scratch    # where the caller's words start
        size = self._more + more
        # (no copies: nothing is launched, and every expert starts at row 0)
        self.buffer = torch.empty(size, dtype=torch.int32, device=device) if n else torch.zeros(size, dtype=torch.int32, device=device)
        self.num_tokens, self.top_k, self.num_experts, self.num_copies = num_tokens, top_k, num_experts, n
        # 128-row tiles that this many copies can fill at most, whatever their experts
        active = n if n < num_experts else num_experts
        self.most_tiles = active + (n - active) // 128
        base = self.buffer.data_ptr()
        rows = base + 12 * e
        # addresses: offsets, tiles, wide_tiles, rows, slots, source, scratch
        self._at = (base, base + 4 * e, base + 8 * e, rows, rows + 4 * n, rows + 8 * n, rows + 12 * n)

    def __reduce__(self):
        raise TypeError("a Plan holds addresses of its buffer: it cannot be copied or pickled, make it again from the choices")

    def _per_expert(self, i: int) -> torch.Tensor:
        e = self.num_experts + 1
        return self.buffer.as_strided((e,), (1,), i * e)

    def _per_copy(self, i: int, shape, strides) -> torch.Tensor:
        return self.buffer.as_strided(shape, strides, 3 * (self.num_experts + 1) + i * self.num_tokens * self.top_k)

    @property
    def offsets(self) -> torch.Tensor:
        """[E + 1] first row of each expert; offsets[E] rows are in use."""
        return self._per_expert(0)

    @property
    def tiles(self) -> torch.Tensor:
        """[E + 1] first 128-row tile of each expert."""
        return self._per_expert(1)

    @property
    def wide_tiles(self) -> torch.Tensor:
        """[E + 1] first 256-row tile of each expert."""
        return self._per_expert(2)

    @property
    def rows(self) -> torch.Tensor:
        """[T, k] row of a copy, -1: not routed."""
        return self._per_copy(0, (self.num_tokens, self.top_k), (self.top_k, 1))

    @property
    def slots(self) -> torch.Tensor:
        """[T, k] row counted with every expert padded to whole 128-row tiles, -1: not routed."""
        return self._per_copy(1, (self.num_tokens, self.top_k), (self.top_k, 1))

    @property
    def source(self) -> torch.Tensor:
        """[T * k] copy of a row, -1 behind the last."""
        return self._per_copy(2, (self.num_tokens * self.top_k,), (1,))


class Routing(NamedTuple):
    weights: torch.Tensor   # [T, k] float32
    experts: torch.Tensor   # [T, k] int32, largest weight first; -1: fewer than k candidates
    plan: Plan


def _matrix(t: torch.Tensor, name: str, rows: int | None = None, cols: int | None = None):
    """Checks ``[rows, cols]`` of a floating type whose rows are contiguous -> (rows, columns, pitch in elements)."""
    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dim() == 2 and t.dtype in _KINDS):
        raise ValueError(f"{name}: expected a CUDA float32 / float16 / bfloat16 matrix")
    have_rows, have_cols = t.shape
    if have_rows > MAX_COPIES or have_cols > MAX_COPIES:
        raise ValueError(f"{name}: expected at most {MAX_COPIES} rows and columns, got {tuple(t.shape)}")
    if (rows is not None and have_rows != rows) or (cols is not None and have_cols != cols):
        raise ValueError(f"{name}: expected shape {(rows, cols)}, got {tuple(t.shape)}")
    pitch, step = t.stride()
    if step != 1 and have_cols > 1:
        raise ValueError(f"{name}: the rows have to be contiguous, got strides {t.stride()}")
    return have_rows, have_cols, pitch if have_rows > 1 else have_cols


def _choices(t: torch.Tensor, name: str, dtype: torch.dtype, shape=None) -> None:
    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dim() == 2 and t.dtype == dtype and t.is_contiguous()):
        raise ValueError(f"{name}: expected a contiguous CUDA {dtype} tensor [T, k]")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name}: expected shape {tuple(shape)}, got {tuple(t.shape)}")


def _same_device(first: torch.Tensor, *others) -> None:
    index = first.get_device()
    for t in others:
        if t is not None and t.get_device() != index:
            raise ValueError(f"all tensors have to be on one device, got {t.device} beside {first.device}")


_ENTRIES: dict = {}     # entry points of the library by name


def _call(entry: str, like: torch.Tensor, *args) -> None:
    """An entry point on the device of ``like`` and torch's current stream there."""
    fn = _ENTRIES.get(entry)
    if fn is None:
        fn = _ENTRIES[entry] = getattr(_lib.load(), entry)
    index = like.get_device()
    if torch._C._cuda_getDevice() == index:
        code = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            code = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if code:
        _lib.check(code, entry)


def _operand(t: torch.Tensor, rows: int, k2: int, L: int, name: str) -> int:
    if t.shape == (rows, k2, L) and t.element_size() == 1 and t.is_cuda:
        a, b, c = t.stride()
        if a == k2 and b == 1 and (L == 1 or c == rows * k2):
            return t.data_ptr()
    return _args.operand_ptr(t, rows, k2, L, name)       # (strides of dimensions of size 1 may be others; else it raises)


def _scales(t: torch.Tensor, rows: int, K: int, L: int, name: str) -> int:
    R, Kb = rows // 128, K // 64
    if t.shape == (32, 4, R, 4, Kb, L) and t.element_size() == 1 and t.is_cuda:
        *inner, outer = t.stride()
        if inner == [16, 4, Kb * 512, 1, 512] and (L == 1 or outer == R * Kb * 512):
            return t.data_ptr()
    return _args.scales_ptr(t, rows, K, L, name)


def _new_operand(like: torch.Tensor, rows: int, tile_rows: int, K: int):
    """An operand ``[rows, K/2, 1]`` and the 6-D swizzled view of the scales of ``tile_rows`` rows, not initialised."""
    R, Kb = tile_rows // 128, K // 64
    return (like.new_empty((rows, K // 2, 1), dtype=torch.float4_e2m1fn_x2),
            like.new_empty_strided((32, 4, R, 4, Kb, 1), (16, 4, Kb * 512, 1, 512, R * Kb * 512), dtype=torch.float8_e4m3fn))


def plan(experts: torch.Tensor, num_experts: int) -> Plan:
    """Sorts the choices ``experts`` [T, k] (int32) stably by expert.  Ids outside [0, num_experts) are not routed; an expert
    may stand in a token more than once."""
    _choices(experts, "experts", torch.int32)
    if not 1 <= num_experts <= MAX_EXPERTS:
        raise ValueError(f"num_experts: expected 1 to {MAX_EXPERTS}, got {num_experts}")
    T, k = experts.shape
    if k > MAX_CHOICES:
        raise ValueError(f"experts: expected at most {MAX_CHOICES} choices for a token, got {k}")
    p = Plan(T, k, num_experts, experts.device)
    if T * k:
        _call("nvfp4_moe_plan", experts, experts.data_ptr(), T, num_experts, k, *p._at)
    return p


def route(logits: torch.Tensor, top_k: int, renormalize: bool = True, mask: torch.Tensor | None = None) -> Routing:
    """The ``top_k`` largest of each row of ``logits`` [T, E], ties to the lowest index, with their softmax weights over
    the chosen entries (``renormalize``) or over all, and the plan of that choice.

    NaN and -inf entries, and the rows of tokens whose ``mask`` [T] (bool) is false, are never chosen and take no part in
    the sum; where fewer than ``top_k`` candidates are left the expert is -1 and the weight 0.  Several +inf entries share
    the whole weight.  The weights do not require gradients: theirs is ``route_backward``."""
    T, E, ld = _matrix(logits, "logits")
    if not 1 <= E <= MAX_EXPERTS:
        raise ValueError(f"logits: expected 1 to {MAX_EXPERTS} experts, got {E}")
    if not 1 <= top_k <= min(E, MAX_CHOICES):
        raise ValueError(f"top_k: expected 1 to {min(E, MAX_CHOICES)}, got {top_k}")
    device = logits.device
    if mask is not None:
        if mask.dtype != torch.bool or mask.shape != (T,) or not mask.is_contiguous():
            raise ValueError(f"mask: expected a contiguous bool tensor of shape {(T,)}")
        _same_device(logits, mask)
    # the weights and the choices lie behind the plan's tables (one allocation: each costs as much as a launch).  `.data`:
    # tensors of their own for autograd, so that weights changed in place do not pass for changed choices or tables
    n = T * top_k
    p = Plan(T, top_k, E, device, 2 * n)
    at = p._more
    weights = p.buffer.view(torch.float32).as_strided((T, top_k), (top_k, 1), at).data
    experts = p.buffer.as_strided((T, top_k), (top_k, 1), at + n).data
    if T:
        address = p._at[0] + 4 * at
        _call("nvfp4_moe_route", logits, logits.data_ptr(), _KINDS[logits.dtype], ld, None if mask is None else mask.data_ptr(),
              T, E, top_k, int(renormalize), address, address + 4 * n, *p._at)
    return Routing(weights, experts, p)


def route_backward(grad_weights: torch.Tensor, logits: torch.Tensor, weights: torch.Tensor, experts: torch.Tensor,
                   renormalize: bool = True) -> torch.Tensor:
    """Gradient of ``route``'s weights with respect to ``logits`` (same type and shape; contiguous), from what ``route``
    took and returned.  Entries that took no part have gradient 0."""
    T, E, ld = _matrix(logits, "logits")
    _choices(experts, "experts", torch.int32)
    k = experts.shape[1]
    if not 1 <= E <= MAX_EXPERTS or not 1 <= k <= min(E, MAX_CHOICES):
        raise ValueError(f"experts: expected 1 to {min(E, MAX_CHOICES)} choices of 1 to {MAX_EXPERTS} experts, got {k} of {E}")
    _choices(experts, "experts", torch.int32, (T, k))
    _choices(weights, "weights", torch.float32, (T, k))
    _choices(grad_weights, "grad_weights", torch.float32, (T, k))
    _same_device(logits, weights, experts, grad_weights)
    out = logits.new_empty((T, E))
    if T:
        _call("nvfp4_moe_route_backward", logits, grad_weights.data_ptr(), logits.data_ptr(), _KINDS[logits.dtype], ld,
              weights.data_ptr(), experts.data_ptr(), T, E, k, int(renormalize), out.data_ptr())
    return out


def dispatch(x: torch.Tensor, plan: Plan) -> torch.Tensor:
    """``x`` [T, H] -> [T * k, H] of the same type: every token's row at the rows of its copies.  The result does not
    require gradients: its gradient is ``dispatch_backward``."""
    T, k = plan.num_tokens, plan.top_k
    _, H, ld = _matrix(x, "x", T)
    _same_device(x, plan.buffer)
    out = x.new_empty((T * k, H))
    if out.numel():
        _call("nvfp4_moe_dispatch", x, x.data_ptr(), _KINDS[x.dtype], ld, plan._at[3], plan._at[0], T,
              plan.num_experts, k, H, out.data_ptr())
    return out


def dispatch_backward(grad_rows: torch.Tensor, plan: Plan) -> torch.Tensor:
    """Gradient of ``dispatch``: ``grad_rows`` [T * k, H] -> [T, H], the sum over each token's copies in fp32."""
    return combine(grad_rows, plan)


def combine(y: torch.Tensor, plan: Plan, weights: torch.Tensor | None = None, dtype: torch.dtype | None = None) -> torch.Tensor:
    """``y`` [T * k, H], rows sorted by expert -> [T, H]: the sum of each token's rows times ``weights`` [T, k] (float32; none:
    the plain sum), in fp32, rounded once to ``dtype`` (default: that of ``y``).  Choices that are not routed add nothing.
    The result does not require gradients: theirs are ``combine_backward``."""
    T, k = plan.num_tokens, plan.top_k
    _, H, ld = _matrix(y, "y", T * k)
    dtype = y.dtype if dtype is None else dtype
    if dtype not in _KINDS:
        raise ValueError(f"dtype: expected float32, float16 or bfloat16, got {dtype}")
    if weights is not None:
        _choices(weights, "weights", torch.float32, (T, k))
    _same_device(y, plan.buffer, weights)
    out = y.new_empty((T, H), dtype=dtype) if k else y.new_zeros((T, H), dtype=dtype)
    if out.numel() and k:
        _call("nvfp4_moe_combine", y, y.data_ptr(), _KINDS[y.dtype], ld, None if weights is None else weights.data_ptr(),
              plan._at[3], T, k, H, out.data_ptr(), _KINDS[dtype])
    return out


def combine_backward(grad_out: torch.Tensor, y: torch.Tensor, plan: Plan, weights: torch.Tensor):
    """Gradients of ``combine`` with weights: ``grad_out`` [T, H] -> (that of ``y``, same type, rows that belong to no copy 0;
    that of ``weights`` [T, k], 0 where a choice is not routed).  The order of a dot product's sum follows from the sizes,
    the types, the alignment of addresses and pitches and the number of SMs."""
    T, k = plan.num_tokens, plan.top_k
    _, H, ldo = _matrix(grad_out, "grad_out", T)
    ld = _matrix(y, "y", T * k, H)[2]
    _choices(weights, "weights", torch.float32, (T, k))
    _same_device(y, grad_out, plan.buffer, weights)
    dy = y.new_empty((T * k, H))
    dw = torch.empty_like(weights) if H else torch.zeros_like(weights)
    if dy.numel():
        _call("nvfp4_moe_combine_backward", y, grad_out.data_ptr(), _KINDS[grad_out.dtype], ldo, y.data_ptr(), _KINDS[y.dtype],
              ld, weights.data_ptr(), plan._at[3], plan._at[0], T, plan.num_experts, k, H, dy.data_ptr(),
              dw.data_ptr())
    return dy, dw


def dispatch_nvfp4(x: torch.Tensor, plan: Plan):
    """``dispatch`` with the rows quantised as ``quantize.quantize_operand`` does: ``x`` [T, K] -> (operand
    ``[T * k, K/2, 1]`` float4_e2m1fn_x2, 6-D swizzled scales of the experts' 128-row tiles, ``plan.most_tiles`` of them).
    Scale bytes of rows that do not exist have no meaning.  K is a multiple of 64."""
    T, k = plan.num_tokens, plan.top_k
    _, K, ld = _matrix(x, "x", T)
    if K % 64 or not K:
        raise ValueError(f"x: the width has to be a multiple of 64, got {K}")
    _same_device(x, plan.buffer)
    packed, scales = _new_operand(x, T * k, plan.most_tiles * 128, K)
    if T * k:
        scratch = _lib.load().nvfp4_moe_dispatch_scratch(T, k, K) if T * k * K >= 1 << 24 else 0
        table = x.new_empty(scratch, dtype=torch.uint8) if scratch else None
        offsets, tiles, _, rows, slots, source, _ = plan._at
        _call("nvfp4_moe_dispatch_nvfp4", x, x.data_ptr(), _KINDS[x.dtype], ld, offsets, tiles, rows, slots, source, T,
              plan.num_experts, k, K, packed.data_ptr(), scales.data_ptr(), table.data_ptr() if scratch else None)
    return packed, scales


def _products(a, sfa, weights, plan: Plan, alpha):
    """Checks the operands of an expert product -> (pointers in the C order, alphas pointer, alpha, R, E, N, K)."""
    R, E = plan.num_copies, plan.num_experts
    if a.dim() != 3 or not a.is_cuda:
        raise ValueError("a: expected the CUDA operand [T * k, K/2, 1] that dispatch_nvfp4 returns")
    K, N = 2 * a.shape[1], weights[0].shape[0]
    if K % 256 or not K:
        raise ValueError(f"a: K has to be a multiple of 256, got {K}")
    if N % 128 or not N:
        raise ValueError(f"b: N has to be a multiple of 128, got {N}")
    ptrs = [_operand(a, R, K // 2, 1, "a"), _scales(sfa, plan.most_tiles * 128, K, 1, "sfa")]
    for i in range(0, len(weights), 2):
        ptrs += [_operand(weights[i], N, K // 2, E, "b"), _scales(weights[i + 1], N, K, E, "sfb")]
    _same_device(a, sfa, *weights, plan.buffer)
    alphas = None
    if isinstance(alpha, torch.Tensor):
        if alpha.dtype != torch.float32 or alpha.shape != (E,) or not alpha.is_contiguous():
            raise ValueError(f"alpha: expected a number or a contiguous float32 tensor of shape {(E,)}")
        _same_device(a, alpha)
        alphas, alpha = alpha.data_ptr(), 1.0
    return ptrs + [*plan._at[:3], alphas], float(alpha), R, E, N, K


def expert_gemm(a, sfa, b, sfb, plan: Plan, alpha=1.0) -> torch.Tensor:
    """``y[r] = fp16(alpha_e * a[r] @ b_e^T)`` for every sorted row r of expert e -> fp16 [T * k, N].  ``a``, ``sfa`` as
    ``dispatch_nvfp4`` or ``expert_dual_gemm_nvfp4`` returns them, ``b`` [N, K/2, E] with its 6-D scales; ``alpha`` a number
    or a float32 tensor [E], the experts' global scales.  N is a multiple of 128, K of 256."""
    ptrs, alpha, R, E, N, K = _products(a, sfa, (b, sfb), plan, alpha)
    c = a.new_empty((R, N), dtype=torch.float16)
    if R:
        _call("nvfp4_moe_gemm", a, *ptrs, c.data_ptr(), R, E, N, K, alpha)
    return c


def expert_dual_gemm(a, sfa, b1, sfb1, b2, sfb2, plan: Plan, alpha=1.0) -> torch.Tensor:
    """``fp16(silu(alpha_e * a[r] @ b1_e^T) * (alpha_e * a[r] @ b2_e^T))`` -> fp16 [T * k, N]; arguments as for
    ``expert_gemm``."""
    ptrs, alpha, R, E, N, K = _products(a, sfa, (b1, sfb1, b2, sfb2), plan, alpha)
    c = a.new_empty((R, N), dtype=torch.float16)
    if R:
        _call("nvfp4_moe_dual_gemm", a, *ptrs, c.data_ptr(), R, E, N, K, alpha)
    return c


def expert_dual_gemm_nvfp4(a, sfa, b1, sfb1, b2, sfb2, plan: Plan, alpha=1.0):
    """``expert_dual_gemm`` with its rows quantised to NVFP4, bit for bit what quantising the fp16 rows gives -> (operand
    ``[T * k, N/2, 1]``, 6-D scales): ``a`` and ``sfa`` of the next product of the same plan, for which N has to be a
    multiple of 256 (it is that product's K)."""
    ptrs, alpha, R, E, N, K = _products(a, sfa, (b1, sfb1, b2, sfb2), plan, alpha)
    packed, scales = _new_operand(a, R, plan.most_tiles * 128, N)
    if R:
        _call("nvfp4_moe_dual_gemm_nvfp4", a, *ptrs, packed.data_ptr(), scales.data_ptr(), R, E, N, K, alpha)
    return packed, scales

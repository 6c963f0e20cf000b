"""Mixtures of experts: the choice of experts, the products of each expert with
its own tokens, and the gradients of both.  No counterpart in the reference.

    weights, indices = og.route(logits, top_k)                     # [tokens, top_k] each
    plan = og.expert_plan(indices, experts)                        # rows in order of their expert
    h = og.expert_gemm(x, w1, plan, gather=True, activation="swiglu")
    y = og.expert_gemm(h, w2, plan)
    out = og.expert_combine(y, weights, plan, residual=x)

As in `gemm`, operands are contiguous CUDA tensors, K is innermost, sums are
float32, and calls are asynchronous on the current stream of the operands'
device.  How many rows each expert gets is known on the device only: nothing
here synchronises, and all calls can be captured into a CUDA graph.

Nothing is recorded for automatic differentiation: results do not require a
gradient, whatever the operands do.  Call the `_backward`s, or wrap a pair of
calls in a `torch.autograd.Function`.
"""

from ctypes import byref

import torch

from . import capi
from .api import overlap

_SCORES = {"softmax": 0, "sigmoid": 1}
_GRADIENT_TYPES = {torch.bfloat16: b"bf16", torch.float16: b"f16"}
_PRODUCT_TYPES = {**_GRADIENT_TYPES, torch.float8_e4m3fn: b"e4m3"}
_ACTIVATIONS = {**capi.ACTIVATIONS, **capi.GATED_ACTIVATIONS}
_PLAN_CHUNK = 8192  # pairs that a plan takes without a workspace
# Up to this many rows per expert the forward product gathers tokens itself; with more, the copy
# engine's pace of some 50 cycles per four gathered rows would set the tile's, and sorting the rows
# first costs less (8 experts, 960 rows each, 4096 x 4096: 660 us gathered in the product, 199 us
# on sorted rows plus 20 us to sort them; 64 experts, two rows each: 66 us either way, without the copy).
_GATHER_IN_PRODUCT = 16


def _expect(label, t, dtype, shape, device):
    """Raise unless `t` is a contiguous CUDA tensor of this dtype and shape."""
    if not (t.shape == shape and t.dtype is dtype and t.device == device and t.is_contiguous() and t.is_cuda):
        raise TypeError(f"{label} must be a contiguous {dtype} {list(shape)} on {device}, got {t.dtype} {list(t.shape)} on {t.device}")


def _apart(label, t, **others):
    """Raise if `t`, which a launch writes, shares memory with a tensor (or None) that it reads or writes too."""
    for name, other in others.items():
        if other is not None and overlap(t, other):
            raise ValueError(f"{label} and {name} share memory")


def _how(logits, top_k, scores, groups, top_groups, group_top, renormalise, scale):
    sigmoid = _SCORES.get(scores)
    if sigmoid is None:
        raise TypeError(f"scores must be one of {list(_SCORES)}, got {scores!r}")
    dtype = capi.ELEMENT_TYPES.get(logits.dtype)
    if dtype is None or not (logits.is_cuda and logits.dim() == 2 and logits.is_contiguous()):
        raise TypeError("logits must be a contiguous 2-D CUDA tensor of float32, bfloat16 or float16")
    tokens, experts = logits.shape
    return capi.OgRoute(tokens, dtype, experts, top_k, sigmoid, groups, top_groups, group_top, bool(renormalise), scale)


def route(logits, top_k, scores="softmax", bias=None, groups=1, top_groups=1, group_top=2, renormalise=True, scale=1.0):
    """Choose `top_k` experts for every token.

    Args:
        logits: `(tokens, experts)` router outputs, float32, bfloat16 or float16,
            at most 1024 experts.  A logit of -inf is never chosen.
        top_k: experts per token, at most 32.
        scores: "softmax" over a token's logits, or "sigmoid" of each.
        bias: float32 `(experts,)` added to the scores for the choice only (load
            balancing); it has no part in the weights.
        groups, top_groups, group_top: the experts lie in `groups` equal runs (at
            most 32); only the `top_groups` runs whose best `group_top` (1 or 2)
            biased scores add up to most are open to the choice.
        renormalise: divide the chosen scores by their sum.
        scale: a factor on the weights.

    Returns:
        `(weights, indices)`, float32 and int32 `(tokens, top_k)`, the best first
        and the lowest index first among equals.  Where a token has fewer than
        `top_k` experts to choose from, the places left have index -1 and weight
        0.  A NaN score ranks first, and its weight is NaN; softmax and `renormalise`
        make all of that token's weights NaN.
    """
    front = capi.front()
    if front is not None:
        done = front.route(logits, top_k, _SCORES.get(scores), bias, groups, top_groups, group_top, bool(renormalise), scale)
        if done is not None:
            return done
    how = _how(logits, top_k, scores, groups, top_groups, group_top, renormalise, scale)
    if bias is not None:
        _expect("bias", bias, torch.float32, (how.experts,), logits.device)
    weights = logits.new_empty((how.tokens, max(top_k, 0)), dtype=torch.float32)
    indices = torch.empty_like(weights, dtype=torch.int32)
    lib = capi.library("mm")
    lib.routing(lib._route, byref(how), logits.data_ptr(), 0 if bias is None else bias.data_ptr(), weights.data_ptr(),
                indices.data_ptr(), logits.get_device())
    return weights, indices


def route_backward(grad_weights, logits, indices, scores="softmax", renormalise=True, scale=1.0):
    """Gradient of the logits, in their dtype, for a gradient of `route`'s weights.

    The choice itself has no gradient: `indices` are those `route` returned, and
    `scores`, `renormalise` and `scale` those it was called with.
    """
    front = capi.front()
    if front is not None:
        done = front.route_backward(grad_weights, logits, indices, _SCORES.get(scores), bool(renormalise), scale)
        if done is not None:
            return done
    how = _how(logits, indices.size(1) if indices.dim() == 2 else 0, scores, 1, 1, 1, renormalise, scale)
    _expect("indices", indices, torch.int32, (how.tokens, how.top_k), logits.device)
    _expect("grad_weights", grad_weights, torch.float32, (how.tokens, how.top_k), logits.device)
    grad = torch.empty_like(logits)
    lib = capi.library("mm")
    lib.routing(lib._route_gradient, byref(how), grad_weights.data_ptr(), logits.data_ptr(), indices.data_ptr(),
                grad.data_ptr(), logits.get_device())
    return grad


class ExpertPlan:
    """Where every (token, choice) pair's row is, in order of the experts.

    Expert e has the rows `offsets[e] .. offsets[e + 1]`, in the order of their
    tokens; `tokens[row]` is a row's token and `positions[t, j]` the row of token
    t's choice j, or -1 for an index outside 0 .. experts - 1.  With such
    indices there are fewer than `rows` rows; what lies behind the last one is
    neither read nor written.  The three int32 tensors are views of one buffer.
    """

    __slots__ = ("experts", "token_count", "top_k", "rows", "device", "_store", "_offsets", "_tokens", "_positions", "_limit",
                 "_native")

    def __init__(self, experts, device, token_count, top_k, store, address):
        self.experts, self.device, self.token_count, self.top_k = experts, device, token_count, top_k
        rows = self.rows = token_count * top_k  # of the tensors in the plan's order
        self._store = store
        # addresses that the launches take: the first rows (and, behind the last of them, how many rows there are) ...
        self._offsets = address
        self._limit = address + 4 * experts
        self._tokens = self._limit + 4
        self._positions = self._tokens + 4 * rows
        self._native = (experts, token_count, top_k, device.index, address)  # ... and what the native host path takes

    @property
    def offsets(self):
        return self._store[:self.experts + 1]

    @property
    def tokens(self):
        return self._store[self.experts + 1:self.experts + 1 + self.rows]

    @property
    def positions(self):
        return self._store[self.experts + 1 + self.rows:].view(self.token_count, self.top_k)


def expert_plan(indices, experts):
    """Sort the (token, choice) pairs by expert.

    Args:
        indices: int32 `(tokens, top_k)`, as `route` returns them; an index outside
            0 .. experts - 1 goes nowhere.
        experts: how many there are, at most 1024.

    Returns:
        An `ExpertPlan`; the same indices always give the same plan.
    """
    front = capi.front()
    if front is not None:
        made = front.expert_plan(indices, experts, _PLAN_CHUNK)
        if made is not None:
            store, address, token_count, top_k = made
            return ExpertPlan(experts, store.device, token_count, top_k, store, address)
    if not (indices.dtype is torch.int32 and indices.is_cuda and indices.dim() == 2 and indices.is_contiguous()):
        raise TypeError("indices must be a contiguous 2-D int32 CUDA tensor")
    if indices.size(1) < 1:
        raise ValueError("indices must name at least one expert per token")
    if not 1 <= experts <= 1024:
        raise ValueError(f"{experts} experts: 1 to 1024 are served")
    store = torch.empty(experts + 1 + 2 * indices.numel(), device=indices.device, dtype=torch.int32)
    plan = ExpertPlan(experts, indices.device, indices.size(0), indices.size(1), store, store.data_ptr())
    workspace = None
    if plan.rows > _PLAN_CHUNK:
        workspace = torch.empty(-(-plan.rows // _PLAN_CHUNK) * experts, device=indices.device, dtype=torch.int32)
    lib = capi.library("mm")
    lib.routing(lib._expert_plan, indices.data_ptr(), plan.token_count, plan.top_k, experts, plan._offsets, plan._tokens,
                plan._positions, 0 if workspace is None else workspace.data_ptr(), indices.get_device())
    return plan


def _check_product(x, w, plan, gather, activation, types):
    """The checks that a product and its gradients share; returns (name, n, k, gated)."""
    name = types.get(x.dtype)
    if name is None:
        raise TypeError(f"x is {x.dtype}: served are {[str(t) for t in types]}")
    if w.dim() != 3:
        raise TypeError(f"w must be [experts, N, K], got {list(w.shape)}")
    experts, n, k = w.shape
    if experts != plan.experts:
        raise ValueError(f"w has {experts} experts and the plan {plan.experts}")
    _expect("x", x, x.dtype, (plan.token_count if gather else plan.rows, k), plan.device)
    _expect("w", w, x.dtype, (experts, n, k), plan.device)
    if activation not in _ACTIVATIONS:
        raise TypeError(f"activation must be one of {[a for a in _ACTIVATIONS if a]}, got {activation!r}")
    gated = activation in capi.GATED_ACTIVATIONS
    multiple = 16 // x.element_size()
    if not n or not k or k % multiple or (gated and n % 16):
        raise ValueError(f"K must be a positive multiple of {multiple} (got {k}) and N positive, a multiple of 16 "
                         f"with a gated activation (got {n})")
    if (x.data_ptr() | w.data_ptr()) % 16:
        raise ValueError("x and w must start on 16-byte boundaries")
    return name, n, k, gated


def expert_gemm(x, w, plan, gather=False, activation=None, alpha=None, out=None, preactivation=None):
    """Every row times its own expert's weights: `out[r] = act(alpha[e] * x[r] @ w[e].T)`.

    Args:
        x: bfloat16, float16 or float8_e4m3fn rows: `(plan.rows, K)` in the plan's
            order, or with `gather` the `(tokens, K)` tokens themselves, each read
            by the experts it is routed to.
        w: `(experts, N, K)` weights of x's dtype; K a multiple of 8 (e4m3: 16).
        plan: from `expert_plan`.
        activation: None, "relu", "gelu", "gelu_tanh", "silu"; or "swiglu" /
            "geglu": `silu(gate) * up` / `gelu(gate) * up`, where the first half of
            an expert's weight rows gives the gate and the second half up; `out` then
            has N / 2 columns.
        alpha: float32 `(experts,)`, a factor on each expert's products (the
            dequantisation scales of fp8 operands).
        out: written instead of a new tensor; x's dtype, bfloat16 for e4m3.  Neither
            it nor `preactivation` may share memory with another tensor of the call.
        preactivation: a `(plan.rows, N)` tensor of `out`'s dtype that receives the
            activation's argument, which `expert_gemm_backward` reads.

    Returns:
        `(plan.rows, N or N / 2)` rows in the plan's order.  Rows behind the plan's
        last are left as they were.
    """
    front = capi.front()
    if front is not None and out is None:
        done = front.expert_gemm(x, w, plan._native, gather, _ACTIVATIONS.get(activation), alpha, preactivation, _GATHER_IN_PRODUCT)
        if done is not None:
            return done
    name, n, k, gated = _check_product(x, w, plan, gather, activation, _PRODUCT_TYPES)
    device, rows = plan.device, plan.rows
    width = n // 2 if gated else n
    own = torch.bfloat16 if x.dtype is torch.float8_e4m3fn else x.dtype
    if out is None:
        out = torch.empty((rows, width), device=device, dtype=own)
    else:
        _expect("out", out, own, (rows, width), device)
        _apart("out", out, x=x, w=w, alpha=alpha, plan=plan._store)
    if preactivation is not None:
        _expect("preactivation", preactivation, own, (rows, n), device)
        _apart("preactivation", preactivation, out=out, x=x, w=w, alpha=alpha, plan=plan._store)
    if alpha is not None:
        _expect("alpha", alpha, torch.float32, (plan.experts,), device)
    if gather and rows > _GATHER_IN_PRODUCT * min(plan.experts, rows):
        x, gather = _sorted_rows(x, plan, k), False
    capi.library("mm").expert_product(
        capi.FORWARD, name, x, w, out, plan.experts, rows, n, k, plan._offsets, plan._tokens if gather else 0,
        plan.token_count, alpha, _ACTIVATIONS[activation], preactivation)
    return out


def _sorted_rows(x, plan, k):
    """The tokens' rows in the plan's order."""
    rows = x.new_empty((plan.rows, k))
    lib = capi.library("mm")
    lib.routing(lib._expert_gather, x.data_ptr(), plan._tokens, plan._limit, rows.data_ptr(), k * x.element_size(), plan.rows,
                x.get_device())
    return rows


def _combine(y, weights, plan, residual, out, n):
    """The launch of `expert_combine`; `weights` None: ones; `y` may be float32."""
    lib = capi.library("mm")
    lib.routing(lib._expert_combine, capi.ELEMENT_TYPES[out.dtype], y.dtype is torch.float32, y.data_ptr(),
                0 if weights is None else weights.data_ptr(), plan._positions, 0 if residual is None else residual.data_ptr(),
                out.data_ptr(), plan.token_count, plan.top_k, n, out.get_device())


def expert_gemm_backward(grad, x, w, plan, gather=False, activation=None, preactivation=None, want=("x", "w"), out_dtype=None):
    """Gradients of `expert_gemm` with 16-bit operands (and no `alpha`).

    With `dz = grad * activation'(preactivation)`, rounded to the operands' type:
    `x`'s gradient is `dz[r] @ w[e]` (with `gather` summed over a token's rows, in
    the order of its choices), `w[e]`'s the sum of `dz[r].T x[r]` over the expert's
    rows, zero for an expert without any.

    Args:
        grad: `(plan.rows, N)` (gated: N / 2) gradient of the output, in the plan's
            order; rows behind the plan's last are not read.
        x, w, plan, gather, activation: as in the forward call; N a multiple of 8.
        preactivation: the tensor the forward call filled; required with an
            activation.
        want: which of "x" and "w" to compute.
        out_dtype: dtype of `w`'s gradient, and without `gather` of `x`'s: the
            operands' (default) or `torch.float32`.

    Returns:
        `(grad_x, grad_w)`, None in the place of what is not wanted.  Without
        `gather` the rows of `grad_x` behind the plan's last are not written.
    """
    front = capi.front()
    if front is not None and (out_dtype is None or out_dtype is x.dtype) and set(want) <= {"x", "w"}:
        done = front.expert_gemm_backward(grad, x, w, plan._native, gather, _ACTIVATIONS.get(activation), preactivation, "x" in want,
                                          "w" in want)
        if done is not None:
            return done
    name, n, k, gated = _check_product(x, w, plan, gather, activation, _GRADIENT_TYPES)
    if n % 8:
        raise ValueError(f"N must be a multiple of 8, got {n}")
    if not set(want) <= {"x", "w"}:
        raise TypeError(f"want names gradients out of 'x' and 'w', got {want!r}")
    if (activation is None) != (preactivation is None):
        raise TypeError("an activation and its preactivation come together")
    if out_dtype not in (None, x.dtype, torch.float32):
        raise TypeError(f"gradients leave as {x.dtype} or torch.float32, not {out_dtype}")
    device, rows = plan.device, plan.rows
    _expect("grad", grad, x.dtype, (rows, n // 2 if gated else n), device)
    if preactivation is not None:
        _expect("preactivation", preactivation, x.dtype, (rows, n), device)
    for label, t in (("grad", grad), ("preactivation", preactivation)):
        if t is not None and t.data_ptr() % 16:
            raise ValueError(f"{label} must start on a 16-byte boundary")
    lib = capi.library("mm")
    # All that the products write is there before the first of them: the weights' gradient, beside the
    # rows', waits for nothing before it writes, so it may not get memory that another thread frees
    # between the two launches while a launch of its own there still reads it.
    grad_x = grad_w = by_row = None
    if "x" in want:
        # a token's rows are added before anything is rounded
        by_row = torch.empty((rows, k), device=device, dtype=torch.float32 if gather else out_dtype or x.dtype)
        grad_x = torch.empty_like(x) if gather else by_row
    if "w" in want:
        grad_w = torch.empty_like(w, dtype=out_dtype or x.dtype)
    dz = grad
    if activation is not None:
        dz = torch.empty_like(preactivation)
        lib.routing(lib._activation_gradient, capi.ELEMENT_TYPES[x.dtype], _ACTIVATIONS[activation], grad.data_ptr(),
                    preactivation.data_ptr(), dz.data_ptr(), 0, 0, plan._limit, rows, n, x.get_device())
    sorted_x = _sorted_rows(x, plan, k) if gather and "w" in want else x
    if "x" in want:
        lib.expert_product(capi.ROWS_GRADIENT, name, dz, w, by_row, plan.experts, rows, n, k, plan._offsets)
    if "w" in want:
        lib.expert_product(capi.WEIGHTS_GRADIENT, name, dz, sorted_x, grad_w, plan.experts, rows, n, k, plan._offsets,
                           beside_previous=by_row is not None)
    if "x" in want and gather:
        _combine(by_row, None, plan, None, grad_x, k)
    return grad_x, grad_w


def expert_combine(y, weights, plan, residual=None, out=None):
    """A token's rows, weighted and summed: `out[t] = residual[t] + sum_j weights[t, j] * y[row of (t, j)]`.

    Args:
        y: bfloat16 or float16 `(plan.rows, N)`, in the plan's order.
        weights: float32 `(tokens, top_k)`.
        plan: from `expert_plan`.  A pair that goes nowhere adds nothing.
        residual: `(tokens, N)` of y's dtype, or None; may be `out`.
        out: written instead of a new tensor; apart from `residual` itself it may
            share memory with no other tensor of the call.

    Returns:
        `(tokens, N)` of y's dtype, summed in float32 in the order of the choices.
    """
    front = capi.front()
    if front is not None and out is None:
        done = front.expert_combine(y, weights, plan._native, residual)
        if done is not None:
            return done
    n = _check_combine(y, weights, plan)
    shape = (plan.token_count, n)
    if residual is not None:
        _expect("residual", residual, y.dtype, shape, plan.device)
    if out is None:
        out = y.new_empty(shape)
    else:
        _expect("out", out, y.dtype, shape, plan.device)
        _apart("out", out, y=y, weights=weights, plan=plan._store)
        if residual is not None and residual.data_ptr() != out.data_ptr():
            _apart("out", out, residual=residual)
    _combine(y, weights, plan, residual, out, n)
    return out


def _check_combine(y, weights, plan):
    """The checks that the combination and its gradient share; returns its columns."""
    if y.dtype not in _GRADIENT_TYPES:
        raise TypeError(f"y is {y.dtype}: bfloat16 and float16 are served")
    if y.dim() != 2 or y.size(1) < 1:
        raise TypeError(f"y must be [rows, N], got {list(y.shape)}")
    n = y.size(1)
    _expect("y", y, y.dtype, (plan.rows, n), plan.device)
    _expect("weights", weights, torch.float32, (plan.token_count, plan.top_k), plan.device)
    return n


def expert_combine_backward(grad, y, weights, plan):
    """Gradients of `expert_combine`: `(grad_y, grad_weights)`.

    `grad_y` (`(plan.rows, N)`, y's dtype) holds `weights[t, j] * grad[t]` in the row
    of (t, j); rows behind the plan's last are not written.  `grad_weights` (float32)
    holds `<grad[t], y[row of (t, j)]>`, 0 for a pair that goes nowhere.  The
    residual's gradient is `grad` itself.
    """
    front = capi.front()
    if front is not None:
        done = front.expert_combine_backward(grad, y, weights, plan._native)
        if done is not None:
            return done
    n = _check_combine(y, weights, plan)
    _expect("grad", grad, y.dtype, (plan.token_count, n), plan.device)
    grad_y, grad_weights = torch.empty_like(y), torch.empty_like(weights)
    lib = capi.library("mm")
    lib.routing(lib._expert_combine_gradient, capi.ELEMENT_TYPES[y.dtype], grad.data_ptr(), y.data_ptr(), weights.data_ptr(),
                plan._positions, grad_y.data_ptr(), grad_weights.data_ptr(), plan.token_count, plan.top_k, n, y.get_device())
    return grad_y, grad_weights

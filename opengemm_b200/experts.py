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
"""

from dataclasses import dataclass

import torch

from . import capi

_SCORES = {"softmax": 0, "sigmoid": 1}
_PRODUCT_TYPES = {torch.bfloat16: b"bf16", torch.float16: b"f16", torch.float8_e4m3fn: b"e4m3"}
_ACTIVATIONS = {**capi.ACTIVATIONS, **capi.GATED_ACTIVATIONS}
_PLAN_CHUNK = 8192  # pairs that a plan takes without a workspace
# Up to this many rows per expert the forward product gathers tokens itself; with more, the copy
# engine's pace of some 50 cycles per four gathered rows would set the tile's, and sorting the rows
# first costs less (8 experts, 960 rows each, 4096 x 4096: 660 us gathered in the product, 199 us
# on sorted rows plus 20 us to sort them; 64 experts, two rows each: 66 us either way, without the copy).
_GATHER_IN_PRODUCT = 16


def _expect(label, t, dtype, shape, device):
    """Raise unless `t` is a contiguous CUDA tensor of this dtype and shape (None: any extent)."""
    if not (t.is_cuda and t.device == device and t.dtype is dtype and t.is_contiguous() and t.dim() == len(shape)
            and all(want is None or want == have for want, have in zip(shape, t.shape))):
        raise TypeError(f"{label} must be a contiguous {dtype} {list(shape)} on {device}, got {t.dtype} {list(t.shape)} on {t.device}"
                        .replace("None", "any"))


def _how(logits, top_k, scores, groups, top_groups, group_top, renormalise, scale):
    if scores not in _SCORES:
        raise TypeError(f"scores must be one of {list(_SCORES)}, got {scores!r}")
    if not (logits.is_cuda and logits.dim() == 2 and logits.is_contiguous() and logits.dtype in capi.ELEMENT_TYPES):
        raise TypeError("logits must be a contiguous 2-D CUDA tensor of float32, bfloat16 or float16")
    return capi.OgRoute(logits.size(0), capi.ELEMENT_TYPES[logits.dtype], logits.size(1), top_k, _SCORES[scores], groups,
                        top_groups, group_top, bool(renormalise), scale)


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
        0.  A NaN logit ranks first and makes its token's weights NaN.
    """
    how = _how(logits, top_k, scores, groups, top_groups, group_top, renormalise, scale)
    if bias is not None:
        _expect("bias", bias, torch.float32, (logits.size(1),), logits.device)
    weights = torch.empty((logits.size(0), top_k), device=logits.device, dtype=torch.float32)
    indices = torch.empty((logits.size(0), top_k), device=logits.device, dtype=torch.int32)
    capi.library("mm").route(how, logits, bias, weights, indices)
    return weights, indices


def route_backward(grad_weights, logits, indices, scores="softmax", renormalise=True, scale=1.0):
    """Gradient of the logits, in their dtype, for a gradient of `route`'s weights.

    The choice itself has no gradient: `indices` are those `route` returned, and
    `scores`, `renormalise` and `scale` those it was called with.
    """
    how = _how(logits, indices.size(1) if indices.dim() == 2 else 0, scores, 1, 1, 1, renormalise, scale)
    _expect("indices", indices, torch.int32, (logits.size(0), None), logits.device)
    _expect("grad_weights", grad_weights, torch.float32, tuple(indices.shape), logits.device)
    grad = torch.empty_like(logits)
    capi.library("mm").route_gradient(how, grad_weights, logits, indices, grad)
    return grad


@dataclass(frozen=True)
class ExpertPlan:
    """Where every (token, choice) pair's row is, in order of the experts.

    Expert e has the rows `offsets[e] .. offsets[e + 1]`, in the order of their
    tokens; `tokens[row]` is a row's token and `positions[t, j]` the row of token
    t's choice j, or -1 for an index outside 0 .. experts - 1.  With such
    indices there are fewer than `rows` rows; what lies behind the last one is
    neither read nor written.
    """

    offsets: torch.Tensor
    tokens: torch.Tensor
    positions: torch.Tensor
    experts: int

    @property
    def rows(self):
        """Rows of the tensors in the plan's order: tokens x top_k."""
        return self.tokens.size(0)


def expert_plan(indices, experts):
    """Sort the (token, choice) pairs by expert.

    Args:
        indices: int32 `(tokens, top_k)`, as `route` returns them; an index outside
            0 .. experts - 1 goes nowhere.
        experts: how many there are, at most 1024.

    Returns:
        An `ExpertPlan`; the same indices always give the same plan.
    """
    if not (indices.is_cuda and indices.dim() == 2 and indices.is_contiguous() and indices.dtype is torch.int32):
        raise TypeError("indices must be a contiguous 2-D int32 CUDA tensor")
    if indices.size(1) < 1:
        raise ValueError("indices must name at least one expert per token")
    pairs, device = indices.numel(), indices.device
    offsets = torch.empty(experts + 1, device=device, dtype=torch.int32)
    tokens = torch.empty(pairs, device=device, dtype=torch.int32)
    positions = torch.empty(indices.shape, device=device, dtype=torch.int32)
    workspace = None
    if pairs > _PLAN_CHUNK:
        workspace = torch.empty(-(-pairs // _PLAN_CHUNK) * experts, device=device, dtype=torch.int32)
    capi.library("mm").expert_plan(indices, experts, offsets, tokens, positions, workspace)
    return ExpertPlan(offsets, tokens, positions, experts)


def _check_product(x, w, plan, gather, activation, types):
    """The checks that a product and its gradients share; returns (name, n, k, gated)."""
    name = _PRODUCT_TYPES.get(x.dtype)
    if name is None or x.dtype not in types:
        raise TypeError(f"x is {x.dtype}: served are {[str(t) for t in types]}")
    if w.dim() != 3:
        raise TypeError(f"w must be [experts, N, K], got {list(w.shape)}")
    experts, n, k = w.shape
    device = plan.offsets.device
    if experts != plan.experts:
        raise ValueError(f"w has {experts} experts and the plan {plan.experts}")
    _expect("x", x, x.dtype, (plan.positions.size(0) if gather else plan.rows, k), device)
    _expect("w", w, x.dtype, (experts, n, k), device)
    if activation not in _ACTIVATIONS:
        raise TypeError(f"activation must be one of {[a for a in _ACTIVATIONS if a]}, got {activation!r}")
    gated = activation in capi.GATED_ACTIVATIONS
    multiple = 16 // x.element_size()
    if not n or not k or k % multiple or (gated and n % 16):
        raise ValueError(f"K must be a positive multiple of {multiple} (got {k}) and N positive, a multiple of 16 "
                         f"with a gated activation (got {n})")
    for label, t in (("x", x), ("w", w)):
        if t.data_ptr() % 16:
            raise ValueError(f"{label} must start on a 16-byte boundary")
    return name, n, k, gated


def expert_gemm(x, w, plan, gather=False, activation=None, alpha=None, out=None, out_dtype=None, preactivation=None):
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
        out: written instead of a new tensor.
        out_dtype: bfloat16 or float16; x's own by default, bfloat16 for e4m3.
        preactivation: a `(plan.rows, N)` tensor of `out`'s dtype that receives the
            activation's argument, which `expert_gemm_backward` reads.

    Returns:
        `(plan.rows, N or N / 2)` rows in the plan's order.  Rows behind the plan's
        last are left as they were.
    """
    name, n, k, gated = _check_product(x, w, plan, gather, activation, tuple(_PRODUCT_TYPES))
    device, rows = x.device, plan.rows
    width = n // 2 if gated else n
    own = torch.bfloat16 if x.dtype is torch.float8_e4m3fn else x.dtype
    if out_dtype not in (None, own):
        raise TypeError(f"{x.dtype} experts write {own}, not {out_dtype}")
    if out is None:
        out = torch.empty((rows, width), device=device, dtype=own)
    else:
        _expect("out", out, own, (rows, width), device)
    if preactivation is not None:
        _expect("preactivation", preactivation, own, (rows, n), device)
    if alpha is not None:
        _expect("alpha", alpha, torch.float32, (plan.experts,), device)
    if gather and rows > _GATHER_IN_PRODUCT * min(plan.experts, rows):
        x, gather = _sorted_rows(x, plan), False
    capi.library("mm").expert_product(
        capi.FORWARD, name, x, w, out, plan.experts, rows, n, k, plan.offsets, plan.tokens if gather else None,
        x.size(0), alpha, _ACTIVATIONS[activation], preactivation)
    return out


def _sorted_rows(x, plan):
    """The tokens' rows in the plan's order."""
    rows = torch.empty((plan.rows, x.size(1)), device=x.device, dtype=x.dtype)
    capi.library("mm").expert_gather(x, plan.tokens, plan.offsets.data_ptr() + 4 * plan.experts, rows)
    return rows


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
        `(grad_x, grad_w)`, None in the place of what is not wanted.
    """
    name, n, k, gated = _check_product(x, w, plan, gather, activation, (torch.bfloat16, torch.float16))
    if n % 8:
        raise ValueError(f"N must be a multiple of 8, got {n}")
    if not set(want) <= {"x", "w"}:
        raise TypeError(f"want names gradients out of 'x' and 'w', got {want!r}")
    if (activation is None) != (preactivation is None):
        raise TypeError("an activation and its preactivation come together")
    if out_dtype not in (None, x.dtype, torch.float32):
        raise TypeError(f"gradients leave as {x.dtype} or torch.float32, not {out_dtype}")
    device, rows = x.device, plan.rows
    _expect("grad", grad, x.dtype, (rows, n // 2 if gated else n), device)
    if preactivation is not None:
        _expect("preactivation", preactivation, x.dtype, (rows, n), device)
    for label, t in (("grad", grad), ("preactivation", preactivation)):
        if t is not None and t.data_ptr() % 16:
            raise ValueError(f"{label} must start on a 16-byte boundary")
    lib = capi.library("mm")
    dz = grad
    if activation is not None:
        dz = torch.empty_like(preactivation)
        lib.activation_gradient(_ACTIVATIONS[activation], grad, preactivation, dz, n,
                                row_limit=plan.offsets.data_ptr() + 4 * plan.experts)
    grad_x = grad_w = None
    if "x" in want:
        # a token's rows are added before anything is rounded
        grad_x = torch.empty((rows, k), device=device, dtype=torch.float32 if gather else out_dtype or x.dtype)
        lib.expert_product(capi.ROWS_GRADIENT, name, dz, w, grad_x, plan.experts, rows, n, k, plan.offsets)
        if gather:
            by_row, grad_x = grad_x, torch.empty_like(x)
            lib.expert_combine(by_row, None, plan.positions, None, grad_x)
    if "w" in want:
        grad_w = torch.empty(w.shape, device=device, dtype=out_dtype or x.dtype)
        sorted_x = _sorted_rows(x, plan) if gather else x
        lib.expert_product(capi.WEIGHTS_GRADIENT, name, dz, sorted_x, grad_w, plan.experts, rows, n, k, plan.offsets)
    return grad_x, grad_w


def expert_combine(y, weights, plan, residual=None, out=None):
    """A token's rows, weighted and summed: `out[t] = residual[t] + sum_j weights[t, j] * y[row of (t, j)]`.

    Args:
        y: bfloat16 or float16 `(plan.rows, N)`, in the plan's order.
        weights: float32 `(tokens, top_k)`.
        plan: from `expert_plan`.  A pair that goes nowhere adds nothing.
        residual: `(tokens, N)` of y's dtype, or None; may be `out`.
        out: written instead of a new tensor.

    Returns:
        `(tokens, N)` of y's dtype, summed in float32 in the order of the choices.
    """
    device = plan.offsets.device
    if y.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"y is {y.dtype}: bfloat16 and float16 are served")
    _expect("y", y, y.dtype, (plan.rows, None), device)
    _expect("weights", weights, torch.float32, tuple(plan.positions.shape), device)
    shape = (plan.positions.size(0), y.size(1))
    if residual is not None:
        _expect("residual", residual, y.dtype, shape, device)
    if out is None:
        out = torch.empty(shape, device=device, dtype=y.dtype)
    else:
        _expect("out", out, y.dtype, shape, device)
    capi.library("mm").expert_combine(y, weights, plan.positions, residual, out)
    return out


def expert_combine_backward(grad, y, weights, plan):
    """Gradients of `expert_combine`: `(grad_y, grad_weights)`.

    `grad_y` (`(plan.rows, N)`, y's dtype) holds `weights[t, j] * grad[t]` in the row
    of (t, j); rows behind the plan's last are not written.  `grad_weights` (float32)
    holds `<grad[t], y[row of (t, j)]>`, 0 for a pair that goes nowhere.  The
    residual's gradient is `grad` itself.
    """
    device = plan.offsets.device
    if y.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"y is {y.dtype}: bfloat16 and float16 are served")
    _expect("y", y, y.dtype, (plan.rows, None), device)
    _expect("weights", weights, torch.float32, tuple(plan.positions.shape), device)
    _expect("grad", grad, y.dtype, (plan.positions.size(0), y.size(1)), device)
    grad_y, grad_weights = torch.empty_like(y), torch.empty_like(weights)
    capi.library("mm").expert_combine_gradient(grad, y, weights, plan.positions, grad_y, grad_weights)
    return grad_y, grad_weights

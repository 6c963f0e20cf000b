"""Definitions in 64 bits of the feed-forward operators, and the tolerances
their results are held to: one rounding to the output type on top of the error
of float32 accumulation, which the tests derive from the operands."""

import torch

HALF_STEP = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16, torch.float32)}
ACTIVATIONS = ["relu", "gelu", "gelu_tanh", "silu"]


def act(name, z):
    """The activation in 64 bits; gated ones take the gate from the first half of the columns."""
    if name in ("swiglu", "geglu"):
        gate, up = z.chunk(2, -1)
        return act("silu" if name == "swiglu" else "gelu", gate) * up
    if name == "relu":
        return torch.relu(z)
    if name == "gelu":
        return z * 0.5 * torch.special.erfc(-z / 2**0.5)
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh((2 / torch.pi) ** 0.5 * (z + 0.044715 * z**3)))
    if name == "silu":
        return z * torch.sigmoid(z)
    return z


def act_gradient(name, z, g):
    """g times the activation's Jacobian, by automatic differentiation in 64 bits."""
    if name is None:
        return g
    z = z.detach().clone().requires_grad_()
    return torch.autograd.grad((act(name, z) * g).sum(), z)[0]


def sum_error(magnitudes, terms):
    """Bound of the error of a float32 sum of `terms` products whose magnitudes add up to
    `magnitudes`: a matrix instruction adds at least eight products at a time and may cut off
    instead of rounding (2^-23 of the running sum, at most `magnitudes`), once more per instruction."""
    return (terms / 8 + 8) * 2.0**-23 * magnitudes


# No activation here is steeper than 1.13 (gelu and silu near 1.4 and 2.4), and none of their
# evaluations is off by more than a few units of float32 in a value of size |z|: two special
# functions at 2^-22, the polynomial of erf at 1.5e-7, products at 2^-24.
STEEPEST = 1.13


def act_error(z, z_error):
    return STEEPEST * z_error + 1e-6 * (z.abs() + z_error)


def assert_within(got, want, error, what=""):
    """`got` is `want` up to `error` (absolute, before rounding) and one rounding to its type."""
    half = HALF_STEP[got.dtype]
    tolerance = half * (want.abs() + error) + error + torch.finfo(got.dtype).tiny
    off = (got.double() - want).abs()
    bad = ~(off <= tolerance)
    if bad.any():
        at = int((off / tolerance).nan_to_num(nan=float("inf")).flatten().argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} values are off; at {at}: got {got.flatten()[at].item()}, "
                             f"want {want.flatten()[at].item()} within {tolerance.flatten()[at].item()}")

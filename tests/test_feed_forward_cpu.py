"""What the feed-forward entry points refuse before they touch a device, and the layout
of their structures: needs no GPU."""

import ctypes
import shutil
import subprocess

import pytest
import torch

import opengemm_b200 as og
from opengemm_b200 import build, capi

SOME = 0x10000  # an address that is never followed


def lib():
    return capi.library("mm")


def refused(code, text, words):
    assert code not in (capi.OG_OK,)
    assert words in text().decode(), text().decode()


def route(**changes):
    fields = dict(tokens=4, dtype=0, experts=16, top_k=2, sigmoid=0, groups=1, top_groups=1, group_top=2, renormalise=1, scale=1.0)
    fields.update(changes)
    return capi.OgRoute(**fields)


@pytest.mark.parametrize("changes,words", [
    (dict(dtype=3), "dtype"), (dict(experts=0), "experts"), (dict(experts=1025, top_k=1), "1024"), (dict(top_k=0), "top_k"), (dict(top_k=33, experts=64), "top_k"),
    (dict(top_k=17), "top_k"), (dict(tokens=-1), "tokens"), (dict(groups=3), "groups"), (dict(groups=64, experts=128), "groups"), (dict(groups=4, top_groups=0), "top_groups"),
    (dict(groups=4, top_groups=5), "top_groups"), (dict(groups=4, group_top=3), "group_top"), (dict(groups=8, top_k=3), "open groups"),
], ids=str)
def test_route_refuses(changes, words):
    how = route(**changes)
    refused(lib()._route(ctypes.byref(how), SOME, 0, SOME, SOME, 0, 0), lib()._routing_error, words)


def test_route_gradient_refuses():
    refused(lib()._route_gradient(ctypes.byref(route(top_k=40, experts=64)), SOME, SOME, SOME, SOME, 0, 0), lib()._routing_error, "top_k")
    refused(lib()._route_gradient(ctypes.byref(route()), 0, SOME, SOME, SOME, 0, 0), lib()._routing_error, "null")
    refused(lib()._route(ctypes.byref(route()), 0, 0, SOME, SOME, 0, 0), lib()._routing_error, "null")


@pytest.mark.parametrize("args,words", [
    ((SOME, 4, 2, 0, SOME, SOME, SOME, 0), "experts"), ((SOME, 4, 2, 1025, SOME, SOME, SOME, 0), "1024"), ((SOME, 4, 0, 8, SOME, SOME, SOME, 0), "too many"),
    ((SOME, 2**31, 8, 8, SOME, SOME, SOME, SOME), "too many"), ((0, 4, 2, 8, SOME, SOME, SOME, 0), "null"), ((SOME, 4, 2, 8, 0, SOME, SOME, 0), "null"),
    ((SOME, 9000, 2, 8, SOME, SOME, SOME, 0), "workspace"),
], ids=str)
def test_plan_refuses(args, words):
    refused(lib()._expert_plan(*args, 0, 0), lib()._routing_error, words)


def test_combine_gather_and_activation_gradient_refuse():
    error = lib()._routing_error
    refused(lib()._expert_combine(0, 0, SOME, SOME, SOME, 0, SOME, 4, 2, 64, 0, 0), error, "dtype")
    refused(lib()._expert_combine(1, 0, SOME, SOME, SOME, 0, SOME, 4, 2, 0, 0, 0), error, "n = 0")
    refused(lib()._expert_combine(1, 0, SOME, SOME, 0, 0, SOME, 4, 2, 64, 0, 0), error, "null")
    refused(lib()._expert_combine_gradient(3, SOME, SOME, SOME, SOME, SOME, SOME, 4, 2, 64, 0, 0), error, "dtype")
    refused(lib()._expert_combine_gradient(1, SOME, SOME, 0, SOME, SOME, SOME, 4, 2, 64, 0, 0), error, "null")
    refused(lib()._expert_gather(SOME, SOME, SOME, SOME, 24, 4, 0, 0), error, "multiple of 16")
    refused(lib()._expert_gather(SOME + 2, SOME, SOME, SOME, 32, 4, 0, 0), error, "16-byte")
    refused(lib()._activation_gradient(0, 1, SOME, SOME, SOME, 0, 0, 0, 4, 64, 0, 0), error, "dtype")
    refused(lib()._activation_gradient(1, 7, SOME, SOME, SOME, 0, 0, 0, 4, 64, 0, 0), error, "activation")
    refused(lib()._activation_gradient(1, 1, SOME, SOME, SOME, 0, 0, 0, 4, 60, 0, 0), error, "eights")
    refused(lib()._activation_gradient(1, 5, SOME, SOME, SOME, SOME, SOME, 0, 4, 64, 0, 0), error, "gated")


def product(**changes):
    fields = dict(x=SOME, w=SOME, offsets=SOME, tokens=0, alpha=0, out=SOME, preactivation=0, mode=0, groups=4, rows=8, x_rows=8, n=64, k=64, activation=0, out_f32=0,
                  factor=1.0, beside_previous=0, dtype=b"bf16")
    fields.update(changes)
    return capi.OgExpertProduct(**fields)


@pytest.mark.parametrize("changes,words", [
    (dict(mode=3), "mode"), (dict(dtype=b"f32"), "dtype"), (dict(dtype=b"e4m3", mode=1), "dtype"), (dict(groups=0), "experts"), (dict(groups=1025), "1024"),
    (dict(offsets=0), "table"), (dict(rows=-1), "rows"), (dict(n=0), "n = 0"), (dict(k=60), "16 bytes"), (dict(dtype=b"e4m3", k=72), "16 bytes"),
    (dict(mode=1, n=60), "16 bytes"), (dict(activation=7), "activation"), (dict(mode=2, activation=1), "activation"), (dict(activation=5, n=72), "16 weight rows"),
    (dict(out_f32=1), "16-bit"), (dict(mode=1, tokens=SOME), "gathers"),
], ids=str)
def test_products_refuse(changes, words):
    refused(lib()._expert_product(ctypes.byref(product(**changes)), 0, 0), lib()._experts_error, words)


def test_product_on_a_device_out_of_range():
    refused(lib()._expert_product(ctypes.byref(product()), 64, 0), lib()._experts_error, "out of range")


@pytest.mark.parametrize("changes,words", [(dict(dtype=b"tf32"), "dtype"), (dict(activation=5), "activation"), (dict(n=60), "eights"), (dict(k=12), "eights"), (dict(m=-1), "m = -1"), (dict(activation=1), "workspace")], ids=str)
def test_gemm_gradients_refuse(changes, words):
    fields = dict(grad=SOME, a=SOME, b=SOME, z=SOME, grad_a=SOME, grad_b=SOME, grad_bias=0, workspace=0, m=8, n=64, k=64, activation=0, out_f32=0, factor=1.0, dtype=b"f16")
    fields.update(changes)
    refused(lib()._gemm_gradients(ctypes.byref(capi.OgGemmGradients(**fields)), 0, 0), lib()._experts_error, words)
    if words != "workspace":
        assert lib()._gradients_workspace(ctypes.byref(capi.OgGemmGradients(**fields)), 0) < 0


def test_gradients_workspace():
    """dz, the bias's sums, and the partial sums of products cut along their reduction."""
    def size(m, n, k, activation=0, bias=0, a=SOME, b=SOME):
        return lib()._gradients_workspace(ctypes.byref(capi.OgGemmGradients(grad_a=a, grad_b=b, grad_bias=bias, m=m, n=n, k=k, activation=activation, dtype=b"bf16")), -1)

    assert size(4096, 8192, 4096) == 0
    assert size(4096, 8192, 4096, activation=1) == 4096 * 8192 * 2
    assert size(4096, 8192, 4096, activation=1, bias=SOME) == 4096 * 8192 * 2 + 64 * 8192 * 4
    few_rows = size(36, 8064, 2680, b=0)
    assert few_rows > 0 and few_rows % (36 * 2680 * 4) == 0  # whole parts of the rows' gradient
    assert size(0, 64, 64, activation=1, bias=SOME) == 0


@pytest.mark.parametrize("name,m,fields,words", [
    ("bf16", 8, dict(activation=5), "activation"), ("bf16", 2, dict(activation=9), "activation"), ("s8", 8, dict(activation=1), "integers"),
    ("bf16", 8, dict(activation=1, preactivation=SOME + 8), "16-byte"), ("bf16", 8, dict(residual=SOME + 2), "element boundary"),
    ("nvfp4", 8, dict(activation=1, out_format=4), "out_format"), ("nvfp4", 8, dict(residual=SOME, out_format=1, out_scales=SOME), "no residual"),
], ids=str)
def test_fused_launch_refuses(name, m, fields, words):
    library, g = capi.bind(name, m, 64, 128, {"output_n": 64})
    epilogue = capi.OgEpilogue(alpha=1.0, **fields)
    scales = SOME if og.DTYPES[name].impl == "smm" else 0
    code = library._fused(ctypes.byref(g), SOME, SOME, scales, scales, SOME, 0, 0, ctypes.byref(epilogue))
    refused(code, library._error, words)


def test_null_structures():
    assert lib()._expert_product(None, 0, 0) != capi.OG_OK
    assert lib()._gemm_gradients(None, 0, 0) != capi.OG_OK
    assert lib()._route(None, SOME, 0, SOME, SOME, 0, 0) != capi.OG_OK
    library, g = capi.bind("bf16", 8, 64, 64, {"output_n": 64})
    assert library._fused(ctypes.byref(g), SOME, SOME, 0, 0, SOME, 0, 0, None) != capi.OG_OK


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs a C compiler")
def test_structures_match_the_header(tmp_path):
    """Sizes and field offsets, as the C compiler lays them out."""
    structures = {"OgEpilogue": capi.OgEpilogue, "OgExpertProduct": capi.OgExpertProduct, "OgRoute": capi.OgRoute, "OgGemmGradients": capi.OgGemmGradients}
    lines = []
    for name, s in structures.items():
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        lines += [f'printf("%zu\\n", offsetof({name}, {f[0]}));' for f in s._fields_]
    source = tmp_path / "sizes.c"
    source.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "opengemm_b200.h"\nint main(void) {\n' + "\n".join(lines) + "\nreturn 0; }\n")
    subprocess.run(["gcc", "-I", str(build.ROOT / "include"), str(source), "-o", str(tmp_path / "sizes")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "sizes")], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for s in structures.values():
        want.append(ctypes.sizeof(s))
        want += [getattr(s, f[0]).offset for f in s._fields_]
    assert got == want


def test_the_native_host_path_leaves_what_it_does_not_serve_to_the_python_one():
    """It answers None, whatever it is given, and the Python front end raises what there is to raise."""
    front = capi.front()
    assert front is not None
    cpu = torch.zeros(4, 8)
    plan = (3, 4, 2, 0, SOME)
    calls = {
        "route": [(cpu, 2, 0, None, 1, 1, 2, 1, 1.0), (None, 2, 0, None, 1, 1, 2, 1, 1.0), ("logits", "2", 0, None, 1, 1, 2, 1, 1.0), ()],
        "route_backward": [(cpu, cpu, cpu.int(), 0, 1, 1.0), (None,) * 6],
        "expert_plan": [(cpu.int(), 3, 8192), (None, 3, 8192), (cpu.int(), "3", 8192)],
        "expert_gemm": [(cpu, cpu, plan, False, 0, None, None, 16), (cpu, cpu, None, False, 0, None, None, 16), (cpu, cpu, (1, 2), False, 0, None, None, 16)],
        "expert_gemm_backward": [(cpu, cpu, cpu, plan, False, 0, None, True, True)],
        "expert_combine": [(cpu, cpu, plan, None), (cpu, cpu, (3, 4, 2, 0, -1), None)],
        "expert_combine_backward": [(cpu, cpu, cpu, plan)],
        "gemm": [(cpu, cpu, None, None, None, None, None, 1, None, None, False), (cpu, None, None, None, torch.bfloat16, 1.0, None, None, None, None, False)],
        "gemm_backward": [(cpu, cpu, cpu, 0, None, None, True, True, True)],
        "learn": [(cpu, cpu, None, None, False, SOME, torch.float32, 0, 0)],
    }
    for name, all_args in calls.items():
        for args in all_args:
            assert getattr(front, name)(*args) is None, (name, args)
    with pytest.raises(RuntimeError, match="missing"):
        front.bind({})
    capi.use_front(True)
    assert capi.front() is not None  # bound again


def test_calls_on_cpu_tensors_are_refused():
    x, w = torch.zeros(8, 64, dtype=torch.bfloat16), torch.zeros(3, 32, 64, dtype=torch.bfloat16)
    with pytest.raises(TypeError):
        og.gemm(x, w[0], activation="relu")
    with pytest.raises(TypeError):
        og.gemm_backward(torch.zeros(8, 32, dtype=torch.bfloat16), x, w[0])
    with pytest.raises(TypeError):
        og.route(torch.zeros(4, 8), 2)
    with pytest.raises(TypeError):
        og.expert_plan(torch.zeros(4, 2, dtype=torch.int32), 3)

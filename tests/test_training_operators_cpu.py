"""What layer norm, the recurrence, the norm over gradients and AdamW behind it refuse, and what they would launch, from their own
host code and without a GPU: the checks are compiled for the host and linked with a runtime that notes launches."""
import ctypes
import math
import os
import subprocess

import pytest
import torch

from adhip import decoder, operators as ops
from adhip.device import library_path

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")


class Checked:
    """As a `HipDevice` whose launches are noted."""

    def __init__(self, lib):
        self._lib, self._ctx = lib, 1

    def last_error(self):
        return self._lib.adhip_last_error(self._ctx).decode()

    def launches(self):
        room = (ctypes.c_uint32 * 400)()
        n = self._lib.noted_launches(room, 100)
        return [tuple(room[4 * i:4 * i + 4]) for i in range(n)]


@pytest.fixture(scope="module")
def dev(tmp_path_factory):
    if not os.path.exists(HIPCC):
        pytest.skip("no hipcc to build the checks with")
    work, csrc = tmp_path_factory.mktemp("checks"), os.path.dirname(library_path())
    objects = []
    steps = []
    for src in [os.path.join(csrc, n + ".hip") for n in ("adamw", "gradients", "layer_norm", "recurrence")] + [
            os.path.join(ROOT, "tests", "cxx", "operator_checks.cpp")]:
        objects.append(str(work / (os.path.basename(src) + ".o")))
        steps.append(subprocess.Popen([HIPCC, "-x", "hip", "--offload-arch=gfx950", "--cuda-host-only", "-std=c++17", "-O1", "-fPIC", "-c", src,
                                       "-o", objects[-1]], stderr=subprocess.PIPE, text=True))
    for s in steps:
        said = s.communicate()[1]
        assert s.returncode == 0, said
    lib = str(work / "checks.so")
    # (each file asks for the device code that a whole build would have put beside it)
    wanted = {x.split()[-1] for x in subprocess.run(["nm", "-u", *objects], check=True, capture_output=True, text=True).stdout.splitlines()
              if "__hip_fatbin" in x}
    subprocess.run(["g++", "-shared", "-o", lib, *objects, "-Wl,-Bsymbolic", *[f"-Wl,--defsym={x}=0" for x in sorted(wanted)]], check=True)
    loaded = ctypes.CDLL(lib)
    loaded.adhip_last_error.argtypes, loaded.adhip_last_error.restype = [ctypes.c_void_p], ctypes.c_char_p
    return Checked(loaded)


class Array:
    """Says where it is and how it lies; there is no memory behind it."""
    is_cuda = True

    def __init__(self, *shape, dtype="float32", stride=None, at=4096):
        self.shape, self.dtype, self._at = tuple(shape), dtype, at
        packed, n = [], 1
        for d in reversed(shape):
            packed.append(n)
            n *= d
        self._stride = tuple(reversed(packed)) if stride is None else tuple(stride)
        self._packed = stride is None
        self.nbytes = n * {"float32": 4, "bfloat16": 2, "int32": 4, "float8_e4m3fn": 1, "float16": 2}[dtype]

    def stride(self):
        return self._stride

    def data_ptr(self):
        return self._at

    def numel(self):
        return math.prod(self.shape)

    def is_contiguous(self):
        return self._packed


ROOM = Array(1 << 26, dtype="int32")


def refused(dev, what, call, *args, **how):
    with pytest.raises((RuntimeError, ValueError), match=what):
        call(dev, *args, **how)
    assert dev.launches() == [], "nothing is queued by a call that is refused"


# ---- layer norm ---------------------------------------------------------------------------------------------------------


def test_layer_norm_refusals(dev):
    x = Array(6, 40)
    good = dict(weight=Array(40), bias=Array(40), stats=Array(6, 2))
    ops.layer_norm(dev, x, x, **good)
    assert len(dev.launches()) == 1
    no = lambda what, *args, **how: refused(dev, what, ops.layer_norm, *args, **{**good, **how})  # noqa: E731
    no("f32 or bf16", Array(6, 40, dtype="int32"), x)
    no("not supported", Array(6, 40, dtype="float16"), x)
    no("1 dims", Array(40), Array(40), stats=None)
    no("elements, 1 to 16384", Array(6, 0), Array(6, 0), weight=None, bias=None)
    no("elements, 1 to 16384", Array(1, 16385), Array(1, 16385), weight=None, bias=None)
    no("too many", Array(1 << 31, 1), Array(1 << 31, 1), weight=None, bias=None, stats=None)
    no("out is", x, Array(6, 41))
    no("out is", x, Array(5, 40))
    no("out is bf16", x, Array(6, 40, dtype="bfloat16"))
    no("out has 3 dims", x, Array(1, 6, 40))
    no("last stride", Array(6, 40, stride=(80, 2)), x)
    no("share memory", x, Array(6, 40, stride=(39, 1)))
    no("share memory", x, Array(6, 40, stride=(0, 1)))
    no("negative stride", Array(6, 40, stride=(-40, 1)), x)
    no("x is missing", Array(6, 40, at=0), x)
    no("aligned", Array(6, 40, at=4098), x)
    no("total has 0 dims", x, x, added=x)
    no("added has 0 dims", x, x, total=x)
    no("added is", x, x, added=Array(6, 41), total=x)
    no("total and out are one array", x, x, added=x, total=x)
    no("weight is", x, x, weight=Array(41))
    no("weight and bias are bf16", x, x, weight=Array(40, dtype="bfloat16"), bias=None)
    no("one type is wanted", x, x, bias=Array(40, dtype="bfloat16"))
    no("weight has 2 dims", x, x, weight=Array(1, 40))
    no("last stride of bias", x, x, bias=Array(40, stride=(2,)))
    no("stats is", x, x, stats=Array(6, 3))
    no("stats is", x, x, stats=Array(5, 2))
    no("stats is", x, x, stats=Array(6, 2, stride=(4, 1)))
    no("stats is int32", x, x, stats=Array(6, 2, dtype="int32"))
    no("8 bytes", x, x, stats=Array(6, 2, at=4100))
    for eps in (0.0, -1e-5, math.nan, math.inf, 1e-60):
        no("eps", x, x, eps=eps)
    wide = Array(6, 40, dtype="bfloat16")
    refused(dev, "one type", ops.layer_norm, wide, wide, weight=Array(40), bias=Array(40, dtype="bfloat16"))


def test_layer_norm_backward_refusals(dev):
    x, stats = Array(6, 40), Array(6, 2)
    need = ops.layer_norm_workspace(dev, x)
    assert need >= 2 * 40 * 4
    good = dict(weight=Array(40), weight_grad=Array(40), bias_grad=Array(40), workspace=ROOM)
    ops.layer_norm_backward(dev, x, stats, x, x, **good)
    assert len(dev.launches()) == 2
    ops.layer_norm_backward(dev, x, stats, x, x, weight=Array(40))
    assert len(dev.launches()) == 1
    no = lambda what, *args, **how: refused(dev, what, ops.layer_norm_backward, *args, **{**good, **how})  # noqa: E731
    no("stats has 0 dims", x, None, x, x)
    no("out_grad is", x, stats, Array(6, 41), x)
    no("x_grad is bf16", x, stats, x, Array(6, 40, dtype="bfloat16"))
    no("share memory", x, stats, x, Array(6, 40, stride=(20, 1)))
    no("total_grad is", x, stats, x, x, total_grad=Array(7, 40))
    no("weight_grad is", x, stats, x, x, weight_grad=Array(39))
    no("bias_grad is int32", x, stats, x, x, bias_grad=Array(40, dtype="int32"))
    no("workspace has 0 bytes", x, stats, x, x, workspace=None)
    no("workspace has", x, stats, x, x, workspace=Array(need - 1, dtype="float8_e4m3fn"))
    no("aligned to 16", x, stats, x, x, workspace=Array(need, dtype="int32", at=4104))
    refused(dev, "elements, 1 to 16384", ops.layer_norm_workspace, Array(3, 20000))
    refused(dev, "in device memory", ops.layer_norm, torch.zeros(6, 40), x)
    refused(dev, "in device memory", ops.layer_norm_backward, x, stats, x, x, workspace=torch.zeros(9))


def test_layer_norm_launches_fit(dev):
    """Workgroups of every size cover the rows, and a workspace holds what each of them leaves."""
    for size in (1, 16, 256, 257, 1024, 1025, 4096, 4097, 16384):
        for rows in (1, 5, 1000, 100000, (1 << 31) - 1):
            for dtype in ("float32", "bfloat16"):
                x = Array(rows, size, dtype=dtype)
                ops.layer_norm(dev, x, x)
                (gx, gy, gz, threads), = dev.launches()
                assert gx * threads < 1 << 32 and (gy, gz) == (1, 1)
                ops.layer_norm_backward(dev, x, Array(rows, 2), x, x, weight_grad=Array(size), workspace=ROOM)
                (gx, _, _, threads), (sx, sy, _, st) = dev.launches()
                assert gx * threads < 1 << 32 and sx * 64 >= size and sy == 2
                assert ops.layer_norm_workspace(dev, x) >= gx * 2 * size * 4


# ---- recurrence ---------------------------------------------------------------------------------------------------------


def test_recurrence_refusals(dev):
    x, state, states = Array(3, 300, 40), Array(3, 40), Array(3, 2, 40)
    good = dict(initial=state, final=state, states=states, lengths=Array(3, dtype="int32"), documents=Array(3, 300, dtype="int32"), workspace=ROOM)
    ops.recurrence(dev, x, x, x, **good)
    assert dev.launches()
    no = lambda what, *args, **how: refused(dev, what, ops.recurrence, *args, **{**good, **how})  # noqa: E731
    no("f32 or bf16", Array(3, 300, 40, dtype="int32"), x, x)
    no("x has 2 dims", Array(300, 40), x, x)
    no("gates is bf16", x, Array(3, 300, 40, dtype="bfloat16"), x)
    no("gates is", x, Array(3, 299, 40), x)
    no("out is", x, x, Array(3, 300, 41))
    no("out has 0 dims", x, x, None)
    no("share memory", x, x, Array(3, 300, 40, stride=(0, 40, 1)))
    no("last stride", x, Array(3, 300, 40, stride=(24000, 80, 2)), x)
    no("negative stride", Array(3, 300, 40, stride=(12000, -40, 1)), x, x)
    no("initial is", x, x, x, initial=Array(3, 41))
    no("initial is bf16", x, x, x, initial=Array(3, 40, dtype="bfloat16"))
    no("final is", x, x, x, final=Array(2, 40))
    no("final share memory", x, x, x, final=Array(3, 40, stride=(0, 1)))
    no("states is", x, x, x, states=Array(3, 3, 40))
    no("states share memory", x, x, x, states=Array(3, 2, 40, stride=(40, 40, 1)))
    no("lengths is", x, x, x, lengths=Array(4, dtype="int32"))
    no("lengths is f32", x, x, x, lengths=Array(3))
    no("documents is", x, x, x, documents=Array(3, 301, dtype="int32"))
    no("documents is f32", x, x, x, documents=Array(3, 300))
    far = Array(3, 300, 40, stride=(1 << 40, (1 << 21) + 1, 1))
    no("2\\^21", far, x, x)
    no("2\\^21", x, far, x)
    no("2\\^21", x, x, far)
    no("extents below", Array(1, 1 << 30, 1), Array(1, 1 << 30, 1), Array(1, 1 << 30, 1))
    refused(dev, "in device memory", ops.recurrence, x, torch.zeros(3, 300, 40), x)


def test_recurrence_backward_refusals(dev):
    x, y, state, states = Array(3, 300, 40), Array(3, 300, 40, at=1 << 20), Array(3, 40), Array(3, 2, 40)
    good = dict(final_grad=state, initial_grad=state, workspace=ROOM)
    ops.recurrence_backward(dev, x, x, states, x, x, y, **good)
    assert dev.launches()
    no = lambda what, *args, **how: refused(dev, what, ops.recurrence_backward, *args, **{**good, **how})  # noqa: E731
    no("one array", x, x, states, x, y, y)
    no("states has 0 dims", x, x, None, x, x, x)
    no("states is", x, x, Array(3, 1, 40), x, x, x)
    no("out_grad is", x, x, states, Array(3, 300, 39), x, x)
    no("x_grad share memory", x, x, states, x, Array(3, 300, 40, stride=(0, 40, 1)), x)
    no("gates_grad is bf16", x, x, states, x, x, Array(3, 300, 40, dtype="bfloat16"))
    no("final_grad is", x, x, states, x, x, y, final_grad=Array(3, 39))
    no("initial_grad share memory", x, x, states, x, x, y, initial_grad=Array(3, 40, stride=(0, 1)))
    far = Array(3, 300, 40, stride=(1 << 40, (1 << 21) + 1, 1))
    no("2\\^21", x, x, states, far, x, y)
    no("2\\^21", x, x, states, x, far, y)
    no("2\\^21", x, x, states, x, y, far)


def test_recurrence_workspaces_and_launches(dev):
    """Few channels over many positions are cut into ranges, whose maps a workspace holds; a call without one is refused.  Both passes
    take what one question said, and launches fit."""
    for dtype in ("float32", "bfloat16"):
        for B, L, C in ((1, 1, 1), (1, 9, 1), (1, 256, 64), (1, 5000, 20), (2, 30000, 300), (1, 100000, 8192), (1, 1 << 20, 1), (4, 3000, 4096),
                        (300, 700, 65), (1 << 20, 20, 33), (70000, 1, 1000), (1, 512, 64)):
            x, states, state = Array(B, L, C, dtype=dtype), Array(B, ops.recurrence_blocks(L), C), Array(B, C)
            need = ops.recurrence_workspace(dev, x, backward=True)
            assert need % 8 == 0 and need <= 256 * 8 * max(B * C, 8192)
            room = Array(need, dtype="float8_e4m3fn") if need else None
            for how in (dict(), dict(documents=Array(B, L, dtype="int32")), dict(factors=True)):
                ops.recurrence(dev, x, x, x, states=states, final=state, workspace=room, **how)
                ops.recurrence_backward(dev, x, x, states, x, x, Array(B, L, C, dtype=dtype, at=1 << 50), workspace=room, **how)
                for gx, gy, gz, threads in dev.launches():
                    assert 1 <= gx * threads < 1 << 32 and (gy, gz) == (1, 1)
    x = Array(1, 5000, 20)
    need = ops.recurrence_workspace(dev, x)
    assert need > 0 and ops.recurrence_workspace(dev, Array(4, 3000, 4096)) == 0
    refused(dev, "workspace has 0 bytes", ops.recurrence, x, x, x)
    refused(dev, "workspace has", ops.recurrence, x, x, x, workspace=Array(need - 1, dtype="float8_e4m3fn"))
    refused(dev, "aligned to 16", ops.recurrence, x, x, x, workspace=Array(need, dtype="int32", at=4104))
    refused(dev, "workspace has 0 bytes", ops.recurrence_backward, x, x, Array(1, 20, 20), x, x, x)
    refused(dev, "too many", ops.recurrence, *[Array(1 << 29, 9, 64, dtype="bfloat16")] * 3)
    refused(dev, "too many", ops.recurrence, *[Array(1 << 29, 1, 1 << 20, dtype="bfloat16")] * 3)


# ---- the norm over gradients --------------------------------------------------------------------------------------------


def test_gradient_refusals(dev):
    gs, norm = [Array(5, 7), Array(9, dtype="bfloat16", at=8192)], Array(1)
    need = ops.gradient_norm_workspace(dev, gs)
    good = dict(limit=1.0, factor=Array(1), workspace=Array(need, dtype="float8_e4m3fn"))
    ops.clip_gradients(dev, gs, norm, **good)
    ops.gradient_norm(dev, gs, norm, **good)
    assert dev.launches()
    no = lambda what, *args, **how: refused(dev, what, ops.clip_gradients, *args, **{**good, **how})  # noqa: E731
    no("not supported", [Array(5, dtype="float16")], norm)
    no("f32 or bf16", [Array(5, dtype="int32")], norm)
    no("packed", [Array(5, 7, stride=(14, 2))], norm)
    no("one f32 number", gs, Array(2))
    no("one f32 number", gs, norm, factor=Array(1, dtype="bfloat16"))
    no("norm is missing", gs, None)
    no("norm is missing", gs, Array(1, at=4098))
    no("1 gradients_out for 2", gs, norm, gradients_out=gs[:1])
    no("own type", gs, norm, gradients_out=[gs[0], Array(9)])
    no("packed elements", gs, norm, gradients_out=[gs[0], Array(8, dtype="bfloat16")])
    no("aligned", [Array(5, at=4098)], norm)
    for limit in (0.0, -1.0, math.nan):
        no("limit", gs, norm, limit=limit)
    for scale in (math.nan, math.inf, 1e300):
        no("grad_scale", gs, norm, grad_scale=scale)
    no("workspace has 0 bytes", gs, norm, workspace=None)
    no("workspace has", gs, norm, workspace=Array(need - 1, dtype="float8_e4m3fn"))
    no("aligned to 8", gs, norm, workspace=Array(need, dtype="int32", at=4100))
    # a list that names a gradient twice, or a part of one
    no("share memory", gs[:1] * 2, norm, workspace=ROOM)
    no("share memory", [Array(100, at=4096), Array(100, at=4096 + 396)], norm, workspace=ROOM)
    ops.clip_gradients(dev, [Array(100, at=4096), Array(100, at=4096 + 400), Array(0, at=4096)], norm, limit=1.0, workspace=ROOM)
    ops.gradient_norm(dev, gs[:1] * 2, norm, workspace=ROOM)
    assert len(dev.launches()) == 2
    # a gradient where another clipped one is written, or where its own one is written a little apart
    x, y, z = Array(100, at=4096), Array(100, at=4496), Array(100, at=4896)
    lies = "lies where another"
    no(lies, [x, y], norm, gradients_out=[y, x], workspace=ROOM)
    no(lies, [x, y], norm, gradients_out=[Array(100, at=8192), x], workspace=ROOM)
    no(lies, [x, x], norm, gradients_out=[z, x], workspace=ROOM)
    no(lies, [x], norm, gradients_out=[Array(100, at=4096 + 4)], workspace=ROOM)
    no(lies, [Array(100, at=4096 + 4)], norm, gradients_out=[x], workspace=ROOM)
    no(lies, [Array(200, at=4096)], norm, gradients_out=[Array(200, at=4496)], workspace=ROOM)
    for outs in ([z, Array(100, at=8192)], [x, z], [z, y]):
        ops.clip_gradients(dev, [x, y], norm, limit=1.0, gradients_out=outs, workspace=ROOM)
        assert len(dev.launches()) == 1
    ops.clip_gradients(dev, [x, x], norm, limit=1.0, gradients_out=[y, z], workspace=ROOM)
    assert len(dev.launches()) == 1
    refused(dev, "in device memory", ops.gradient_norm, [torch.zeros(3)], norm, workspace=ROOM)
    refused(dev, "in device memory", ops.gradient_norm, gs, torch.zeros(1), workspace=ROOM)
    refused(dev, "in device memory", ops.clip_gradients, gs, norm, limit=1.0, gradients_out=[torch.zeros(5, 7), gs[1]], workspace=ROOM)


def test_gradient_launches_fit(dev):
    many = [Array(1 + 300 * i, at=4096 + (i << 21)) for i in range(1000)]
    room = Array(ops.gradient_norm_workspace(dev, many), dtype="float8_e4m3fn")
    ops.clip_gradients(dev, many, Array(1), limit=1.0, workspace=room)
    seen = dev.launches()
    assert len(seen) <= 2 * 8 + 1 and all(x * t < 1 << 32 for x, _, _, t in seen)
    huge = [Array(1 << 37)]
    ops.gradient_norm(dev, huge, Array(1), workspace=Array(ops.gradient_norm_workspace(dev, huge), dtype="float8_e4m3fn"))
    assert all(x * t < 1 << 32 for x, _, _, t in dev.launches())
    refused(dev, "elements", ops.gradient_norm_workspace, [Array(1 << 50)])


def test_adamw_factor_refusals(dev):
    one = [Array(40)]
    how = dict(step=1, rate=0.1)
    ops.adamw(dev, one, one, one, one, factor=Array(1), **how)
    assert len(dev.launches()) == 1
    refused(dev, "one f32 number", ops.adamw, one, one, one, one, factor=Array(2), **how)
    refused(dev, "one f32 number", ops.adamw, one, one, one, one, factor=Array(1, dtype="int32"), **how)
    refused(dev, "aligned", ops.adamw, one, one, one, one, factor=Array(1, at=4098), **how)
    refused(dev, "in device memory", ops.adamw, one, one, one, one, factor=torch.ones(1), **how)


def test_the_decoder_names_its_layers():
    with pytest.raises(SystemExit, match="attention or recurrence"):
        decoder.main("convolution")


# ---- without a context, and the C structs ---------------------------------------------------------------------------------


def test_calls_without_a_context_or_arguments_are_errors(dev):
    lib = ops._declared(dev._lib)
    for name in ("adhip_layer_norm", "adhip_layer_norm_backward", "adhip_recurrence", "adhip_recurrence_backward", "adhip_gradient_norm",
                 "adhip_clip_gradients"):
        assert getattr(lib, name)(None, bytes(2000), None) != 0 and getattr(lib, name)(1, None, None) != 0
    need = ctypes.c_size_t()
    assert lib.adhip_adamw_scaled(None, bytes(200), None, None) != 0 and lib.adhip_adamw_scaled(1, None, None, None) != 0
    assert lib.adhip_layer_norm_workspace(1, None, ctypes.byref(need)) != 0 and lib.adhip_layer_norm_workspace(1, bytes(2000), None) != 0
    assert lib.adhip_recurrence_workspace(1, None, 0, ctypes.byref(need)) != 0 and lib.adhip_gradient_norm_workspace(1, None, ctypes.byref(need)) != 0
    assert dev.launches() == []


def test_packed_arguments_have_the_layout_of_the_header(tmp_path):
    src = tmp_path / "layout.c"
    src.write_text('''#include "adhip.h"
#include <stdio.h>
#define S(t) printf("%zu\\n", sizeof(t))
#define O(t, f) printf("%zu\\n", offsetof(t, f))
int main(void) {
    S(adhip_layer_norm_args); O(adhip_layer_norm_args, stats); O(adhip_layer_norm_args, out_grad); O(adhip_layer_norm_args, eps);
    O(adhip_layer_norm_args, workspace_bytes); S(adhip_recurrence_args); O(adhip_recurrence_args, documents); O(adhip_recurrence_args, out_grad);
    O(adhip_recurrence_args, factors); O(adhip_recurrence_args, workspace_bytes); S(adhip_gradient); O(adhip_gradient, type);
    S(adhip_gradients_args); O(adhip_gradients_args, limit); O(adhip_gradients_args, norm); O(adhip_gradients_args, workspace_bytes);
    printf("%d\\n", ADHIP_RECURRENCE_BLOCK);
    return 0;
}''')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    c = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    a = ops._ARRAY.size
    assert c == [12 * a + ops._NORM_TAIL.size, 6 * a, 7 * a, 12 * a, 12 * a + 24, 13 * a + ops._RECURRENCE_TAIL.size, 7 * a, 8 * a, 13 * a, 13 * a + 16,
                 32, 24, ops._GRADIENTS.size, 16, 32, 56, ops.RECURRENCE_BLOCK]

"""What of the operators on device arrays can be checked without a GPU: the layout of the C structs that the Python side
packs, the rotary tables, and calls without a context."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

from adhip import operators as ops
from adhip.device import library_path, load_library

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_packed_arguments_have_the_layout_of_the_header(tmp_path):
    src = tmp_path / "layout.c"
    src.write_text('''#include "adhip.h"
#include <stdio.h>
#define S(t) printf("%zu\\n", sizeof(t))
#define O(t, f) printf("%zu\\n", offsetof(t, f))
int main(void) {
    S(adhip_array); O(adhip_array, dims); O(adhip_array, strides); S(adhip_rotary_args); O(adhip_rotary_args, inverse);
    S(adhip_adamw_tensor); O(adhip_adamw_tensor, p_out); O(adhip_adamw_tensor, count); S(adhip_adamw_args); O(adhip_adamw_args, step);
    O(adhip_adamw_args, grad_scale); S(adhip_attention_args); O(adhip_attention_args, slopes); O(adhip_attention_args, out_grad);
    O(adhip_attention_args, scale); O(adhip_attention_args, causal); O(adhip_attention_args, window); O(adhip_attention_args, workspace_bytes);
    return 0;
}''')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    c = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    a = ops._ARRAY.size
    mine = [a, 16, 48, 7 * a + ops._ROTARY_TAIL.size, 7 * a + 4, 12 * 8, 6 * 8, 11 * 8, ops._ADAMW.size, 28, 72,
            14 * a + ops._ATTENTION_TAIL.size, 5 * a, 10 * a, 14 * a, 14 * a + 8, 14 * a + 16, 14 * a + 32]
    assert c == mine


def test_calls_without_a_context_are_errors():
    lib = ops._declared(load_library())
    for call in (lambda: lib.adhip_rotary(None, bytes(600), None), lambda: lib.adhip_attention(None, bytes(1200), None),
                 lambda: lib.adhip_attention_backward(None, bytes(1200), None), lambda: lib.adhip_adamw(None, bytes(100), None),
                 lambda: lib.adhip_sync(None), lambda: lib.adhip_alloc(None, 4, ctypes.byref(ctypes.c_void_p()))):
        assert call() != 0
    assert b"context" in lib.adhip_last_error(None)
    assert lib.adhip_stream(None) is None
    assert os.path.exists(library_path())


def test_rotary_table():
    cos, sin = ops.rotary_table(1000, 64)
    assert cos.shape == sin.shape == (1000, 32) and cos.dtype == np.float32
    at, i = 777, 5
    angle = at * 10000.0 ** (-2 * i / 64)
    assert abs(float(cos[at, i]) - np.cos(angle)) <= 2.0 ** -24 and abs(float(sin[at, i]) - np.sin(angle)) <= 2.0 ** -24
    # angles to the table's last bit far out, where position times frequency in 32 bits is off by hundredths
    far, _ = ops.rotary_table(200001, 8)
    assert abs(float(far[200000, 0]) - np.cos(200000.0)) <= 2.0 ** -24


def test_rotary_table_scaled_for_long_contexts():
    plain, _ = ops.rotary_table(400, 64)
    linear, _ = ops.rotary_table(400, 64, factor=4.0, scaling="linear")
    assert np.array_equal(linear[396], plain[99])
    # by the base: the fastest pair is left alone, the slowest one turns as far as the plain one does at a fourth of the position
    base, _ = ops.rotary_table(400, 64, factor=4.0, scaling="base")
    assert np.array_equal(base[:, 0], plain[:, 0]) and np.allclose(base[396, -1], plain[99, -1], atol=1e-7)
    # in parts: fast pairs are left alone, slow ones are divided, those between are between
    parts, _ = ops.rotary_table(400, 64, factor=4.0, scaling="parts", trained=100)
    per = 10000.0 ** (-np.arange(0, 64, 2) / 64)
    turns = 100 * per / (2 * np.pi)
    assert turns.max() < 32 and (turns < 1).any()
    assert np.array_equal(parts[396, turns < 1], plain[99, turns < 1])
    parts, _ = ops.rotary_table(400, 64, factor=4.0, scaling="parts", trained=100000)
    turns = 100000 * per / (2 * np.pi)
    assert np.array_equal(parts[:, turns > 32], plain[:, turns > 32]) and (turns > 32).any()
    for bad in (dict(rows=0, features=8), dict(rows=4, features=7), dict(rows=4, features=8, base=0.0), dict(rows=4, features=8, scaling="none"),
                dict(rows=4, features=8, scaling="parts"), dict(rows=4, features=2, scaling="base"), dict(rows=4, features=8, factor=0.0)):
        with pytest.raises(ValueError):
            ops.rotary_table(**bad)

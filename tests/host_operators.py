"""Runs hand-written operators on the host, kernels and all: their source compiles as ordinary C++ with a stand-in for HIP
(cxx/host_hip) under which a workgroup's threads run as contexts of one thread, and workgroups one after the other in the order of their
numbers or in the opposite one.  What depends on the order in which workgroups run, and what an access touches, shows here without a GPU."""
import os
import re
import subprocess

import ctypes
import numpy as np
import torch

from adhip.device import library_path

CLANG = "/opt/rocm/lib/llvm/bin/clang++"
HERE = os.path.dirname(os.path.abspath(__file__))


class HostLibrary:
    """Knows the entry points of the sources that it was built from; of others it has a name alone."""

    def __init__(self, lib):
        self._lib, self._others = lib, {}

    def __getattr__(self, name):
        try:
            return getattr(self._lib, name)
        except AttributeError:
            return self._others.setdefault(name, type("Absent", (), {})())


class HostDevice:
    """As a `HipDevice`, of the host."""

    def __init__(self, lib):
        self._lib, self._ctx = HostLibrary(lib), 1

    def last_error(self):
        return self._lib.adhip_last_error(self._ctx).decode()

    def in_both_orders(self, f):
        """What f gives with workgroups in the order of their numbers, and with the last one first."""
        results = []
        for last_first in (0, 1):
            self._lib.host_last_workgroup_first(last_first)
            results.append(f())
        self._lib.host_last_workgroup_first(0)
        return results


class HostArray:
    """A CPU tensor that operators take for an array on their device."""
    is_cuda = True

    def __init__(self, t):
        self.t, self.shape, self.dtype = t, t.shape, t.dtype
        self.nbytes = t.numel() * t.element_size()

    def stride(self):
        return self.t.stride()

    def data_ptr(self):
        return self.t.data_ptr()

    def numel(self):
        return self.t.numel()

    def is_contiguous(self):
        return self.t.is_contiguous()


def build(work, *names):
    """A device whose operators are those of csrc/<name>.hip."""
    csrc, objects, steps = os.path.dirname(library_path()), [], []
    flags = ["-x", "c++", "-std=c++17", "-O2", "-march=native", "-ffp-contract=off", "-fPIC", "-w", "-I", os.path.join(HERE, "cxx", "host_hip"), "-I", csrc]
    for name in names:
        src = os.path.join(work, name + ".cpp")
        with open(os.path.join(csrc, name + ".hip")) as f:
            text = f.read()
        with open(src, "w") as f:  # (statements that hold a value in registers say nothing to the host)
            f.write(re.sub(r"\basm( volatile)?\([^;]*\);", ";", text))
        steps.append(src)
    steps.append(os.path.join(HERE, "cxx", "host_operators.cpp"))
    running = []
    for src in steps:
        objects.append(os.path.join(work, os.path.basename(src) + ".o"))
        running.append(subprocess.Popen([CLANG, *flags, "-c", src, "-o", objects[-1]], stderr=subprocess.PIPE, text=True))
    for r in running:
        said = r.communicate()[1]
        assert r.returncode == 0, said
    lib = os.path.join(work, "host_operators.so")
    subprocess.run([CLANG, "-shared", "-o", lib, *objects, "-Wl,-Bsymbolic"], check=True)
    loaded = ctypes.CDLL(lib)
    loaded.adhip_last_error.argtypes, loaded.adhip_last_error.restype = [ctypes.c_void_p], ctypes.c_char_p
    return HostDevice(loaded)


def seen(t):
    return None if t is None else HostArray(t)


def room(bytes_wanted):
    """A workspace that begins at a multiple of 16, filled with what must not matter."""
    t = torch.from_numpy(np.full(bytes_wanted + 32, 255, np.uint8))
    off = -t.data_ptr() % 16
    return HostArray(t[off:off + bytes_wanted])

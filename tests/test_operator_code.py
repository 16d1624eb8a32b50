"""What the compiled kernels of the operators on device arrays (csrc/*.hip) must keep to, read from the AMD assembly of the
library as it was built: rules of the instruction set that the compiler does not see to inside of inline assembly."""
import os
import re
import subprocess

import pytest

from adhip.device import library_path

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"


@pytest.fixture(scope="module")
def instructions(tmp_path_factory):
    """Every kernel of the library: {name: [instruction text]}, in the order of the code."""
    if not os.path.exists(OBJDUMP):
        pytest.skip("no llvm-objdump to read the library with")
    work = tmp_path_factory.mktemp("code")
    os.symlink(library_path(), work / "library.so")
    subprocess.run([OBJDUMP, "--offloading", "library.so"], cwd=work, check=True, stdout=subprocess.DEVNULL)
    kernels = {}
    for part in sorted(work.glob("*gfx950*")):
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", str(part)], check=True, capture_output=True, text=True).stdout
        body = None
        for line in text.splitlines():
            head = re.match(r"[0-9a-f]+ <(\S+)>:", line)
            if head:
                body = kernels.setdefault(head.group(1), [])
            elif body is not None and line.startswith("\t"):
                body.append(line.split("//")[0].strip())
    return kernels


def scalars(operand):
    """Numbers of the scalar registers that an operand names."""
    m = re.match(r"s\[(\d+):(\d+)\]$|s(\d+)$", operand)
    if not m:
        return set()
    return {int(m.group(3))} if m.group(3) else set(range(int(m.group(1)), int(m.group(2)) + 1))


def operands(text):
    return [x.strip() for x in text.split(None, 1)[1].split(",")] if " " in text else []


def to_lds(text):
    return text.startswith("buffer_load") and text.endswith(" lds")


def test_loads_to_lds_wait_for_their_descriptors(instructions):
    """A vector instruction's result in a scalar register may be read by a memory instruction five wait states later: an
    instruction is one, `s_nop n` is n + 1.  The hardware does not hold the reader back."""
    loads, early = 0, []
    for name, body in instructions.items():
        for i, text in enumerate(body):
            if not to_lds(text):
                continue
            loads += 1
            reads = set().union(*(scalars(x.split()[0]) for x in operands(text)))
            waited, at = 0, i - 1
            while at >= 0 and waited < 5 and reads:
                before = body[at]
                writes = scalars(operands(before)[0].split()[0]) if operands(before) else set()
                if before.startswith("v_") and writes & reads:
                    early.append(f"{name}: {before}; {waited} wait states; {text}")
                    break
                reads -= writes if before.startswith("s_") and not before.startswith(("s_cmp", "s_bitcmp")) else set()
                waited += int(operands(before)[0], 0) + 1 if before.startswith("s_nop") else 1
                at -= 1
    assert loads > 1000, "the kernels of attention bring their tiles to LDS this way"
    assert not early, f"{len(early)} loads of {loads} read a descriptor too early, the first: {early[0]}"


def test_the_join_of_ranges_stays_within_its_sums(tmp_path):
    """Every thread of the joining kernel that adds up reads sums of its own row, and none behind the last thread's, for every
    width and number of ranges.  The kernel's own indices, run on the host."""
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    if not os.path.exists(hipcc):
        pytest.skip("no hipcc to build the indices with")
    src = tmp_path / "join.hip"
    src.write_text('''#include <cstdio>
#include "operator_attention_forward.hpp"
using namespace adhip::attn;
int main() {
    long outside = 0, foreign = 0, left_over = 0;
    for (int D = 1; D <= 256; ++D)
        for (int splits = kFewRanges + 1; splits <= 256; ++splits) {
            const JoinShape j(D, splits);
            if (j.rows < 1 || j.rows * splits > 2048 || j.rows * j.pieces * j.groups > 256) return 1;
            for (int rows = 1; rows <= j.rows; rows += j.rows > 1 ? j.rows - 1 : 1)
                for (int tid = 0; tid < 256; ++tid) {
                    const JoinPlace place(j, rows, tid);
                    left_over += place.row >= j.rows;
                    if (!place.adds()) continue;
                    for (int i = 1; i < j.groups; ++i) {
                        const JoinPlace other(j, rows, tid + i * j.pieces);
                        outside += tid + i * j.pieces >= 256;
                        foreign += other.row != place.row || other.group != i || other.d != place.d;
                    }
                }
        }
    printf("%ld %ld %d\\n", outside, foreign, left_over > 0);
    return 0;
}''')
    csrc = os.path.dirname(library_path())
    exe = tmp_path / "join"
    subprocess.run([hipcc, "--offload-arch=gfx950", "-std=c++17", "-O1", "--cuda-host-only", "-I", csrc, str(src), "-o", str(exe)], check=True,
                   capture_output=True)
    done = subprocess.run([str(exe)], capture_output=True, text=True)
    assert (done.returncode, done.stdout.split()) == (0, ["0", "0", "1"])

"""Wait states around inline assembly, in the machine code of the built library.

The compiler counts the wait states that gfx950 asks for between two instructions, but not where one of
them is inline assembly: those are kept by the sources, and looked for here in what was built from
them, on every path of at most the wanted length.
"""

import re
import shutil
import struct
import subprocess
from pathlib import Path

import pytest

from ninetoothed_amd import _build, _lib

MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"


def _objdump():
    beside = Path(_build.hipcc()).resolve().parent.parent
    for found in (shutil.which("llvm-objdump"), beside / "llvm/bin/llvm-objdump", beside / "bin/llvm-objdump",
                  Path("/opt/rocm/llvm/bin/llvm-objdump")):
        if found and Path(found).exists():
            return str(found)
    pytest.skip("no llvm-objdump in this toolchain")


def _code_objects(data):
    """The gfx950 code objects of the offload bundles in a host library, one a source file."""
    at = data.find(MAGIC)
    while at >= 0:
        (count,) = struct.unpack_from("<Q", data, at + len(MAGIC))
        p = at + len(MAGIC) + 8
        for _ in range(count):
            offset, size, name = struct.unpack_from("<QQQ", data, p)
            target = data[p + 24:p + 24 + name]
            p += 24 + name
            if size and target.endswith(_build.OFFLOAD_ARCH.encode()):
                yield data[at + offset:at + offset + size]
        at = data.find(MAGIC, at + len(MAGIC))


class Kernel:
    """A function's instructions (mnemonic, operands) in order, and where its labels are."""

    def __init__(self, name):
        self.name, self.code, self.labels = name, [], {}

    def behind(self, i, states):
        """Yields (mnemonic, operands, wait states since i) of what may be issued less than ``states`` wait states behind
        instruction i, path by path; a true value sent back ends the path."""
        todo, seen = [(i + 1, 0)], set()
        while todo:
            j, passed = todo.pop()
            while passed < states and j < len(self.code) and (j, passed) not in seen:
                seen.add((j, passed))
                mnemonic, operands = self.code[j]
                j += 1
                if mnemonic == "s_nop":
                    passed += int(operands[0], 0)
                elif mnemonic == "s_endpgm":
                    break
                elif mnemonic == "s_branch" or mnemonic.startswith("s_cbranch"):
                    todo.append((self.labels[operands[0].strip("<>")], passed + 1))
                    if mnemonic == "s_branch":
                        break
                elif (yield mnemonic, operands, passed):
                    break
                passed += 1


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    _lib.load()
    tool, found = _objdump(), []
    for i, obj in enumerate(_code_objects(_build.LIBRARY_PATH.read_bytes())):
        path = tmp_path_factory.mktemp("code") / f"{i}.co"
        path.write_bytes(obj)
        text = subprocess.run([tool, "-d", "--no-show-raw-insn", "--no-leading-addr", "--symbolize-operands", str(path)],
                              check=True, capture_output=True, text=True).stdout
        for line in text.splitlines():
            line = line.split("//")[0].strip()
            label = re.fullmatch(r"(?:[0-9a-f]+ )?<(.+)>:", line)
            if label and re.fullmatch(r"L\d+", label[1]):
                found[-1].labels[label[1]] = len(found[-1].code)
            elif label:
                found.append(Kernel(label[1]))
            elif line and found and not line.startswith("Disassembly") and "file format" not in line:
                mnemonic, _, rest = line.partition(" ")
                found[-1].code.append((mnemonic, re.split(r"[, ]+", rest.strip()) if rest else []))
    assert len(found) > 100 and any("prompt_stream_kernel" in k.name for k in found)
    return found


def registers(operand):
    """The registers that an operand names, as (kind, number)."""
    m = re.fullmatch(r"[-|]*([sva])(?:(\d+)|\[(\d+):(\d+)\])\|?", operand)
    if not m:
        return {operand} if operand in ("vcc", "m0") else set()
    first, last = (m[2], m[2]) if m[2] else (m[3], m[4])
    return {(m[1], n) for n in range(int(first), int(last) + 1)}


def violations(kernels, writes, states, reads):
    """Where an instruction that ``reads`` something is issued less than ``states(mnemonic)`` behind one that
    ``writes`` it (each gives an instruction's registers)."""
    bad = []
    for kernel in kernels:
        for i, (mnemonic, operands) in enumerate(kernel.code):
            live = writes(mnemonic, operands)
            if not live:
                continue
            walk, end = kernel.behind(i, states(mnemonic)), None
            while True:
                try:
                    m, ops, passed = walk.send(end)
                except StopIteration:
                    break
                end = bool(live & reads(m, ops))
                if end:
                    bad.append((kernel.name, f"{mnemonic} {' '.join(operands)}", f"{m} {' '.join(ops)}", passed))
    return bad


def test_a_load_into_lds_comes_a_wait_state_after_its_address(kernels):
    # A load whose data goes to LDS takes the place from M0, one wait state after a scalar instruction wrote it.
    into_lds = [k for k in kernels if any("lds" in ops for _, ops in k.code)]
    assert len(into_lds) > 20
    bad = violations(into_lds, lambda m, ops: {"m0"} if m.startswith("s_") and ops and ops[0] == "m0" else set(),
                     lambda m: 1, lambda m, ops: {"m0"} if "lds" in ops or "load_lds" in m else set())
    assert not bad, (len(bad), bad[:3])


def test_a_load_comes_five_wait_states_after_a_vector_instruction_wrote_its_scalars(kernels):
    # v_readfirstlane and comparisons write scalar registers that a memory instruction reads five wait states later.
    def written(m, ops):
        return {r for r in registers(ops[0]) if r[0] == "s" or r == "vcc"} if m.startswith("v_") and ops else set()

    def read(m, ops):
        if not m.startswith(("buffer_", "global_", "flat_", "scratch_")):
            return set()
        return {r for op in ops for r in registers(op)}

    bad = violations(kernels, written, lambda m: 5, read)
    assert not bad, (len(bad), bad[:3])


def test_inline_assembly_reads_products_when_they_are_there(kernels):
    # A 32 x 32 x 16 product's registers may be read twelve wait states after it, those of 16 x 16 x 32 eight; in the
    # kernels around the cache, inline assembly takes maxima of scores.
    def accumulators(m, ops):
        return registers(ops[0]) if m.startswith("v_mfma") else set()

    def read(m, ops):
        if m.startswith("v_mfma") or not m.startswith(("v_", "ds_", "buffer_", "global_", "scratch_")):
            return set()
        return {r for op in ops for r in registers(op)}

    mine = [k for k in kernels if "prompt_" in k.name or "cache_" in k.name]
    assert len(mine) > 20
    bad = violations(mine, accumulators, lambda m: 12 if "32x32x16" in m else 8, read)
    assert not bad, (len(bad), bad[:3])

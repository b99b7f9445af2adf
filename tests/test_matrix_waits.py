"""The built library's own instructions, read back: on every way through a kernel there are the wait states between a matrix instruction and what reads or
overwrites its result, between a vector instruction and a matrix instruction that takes what it writes, and between one that writes scalar registers and a memory request that
takes them.  None is waited for by the hardware; the compiler fills in what it sees, but it may look at the longer one of two ways that meet, and does not look into assembly.

A wait state is an instruction's slot.  A result needs its matrix instruction's passes (of four cycles) and two more states, of types below 32 bits four more; matrix
instructions follow each other when the one before has made its passes.  A matrix instruction's operand needs two, a scalar register five."""

import heapq
import os
import pathlib
import re
import struct
import subprocess
from concurrent.futures import ProcessPoolExecutor

import pytest

LIBRARY = pathlib.Path(__file__).resolve().parent.parent / "distdl_amd" / "libdistdl_hip.so"
OBJDUMP = pathlib.Path(os.environ.get("ROCM_PATH", "/opt/rocm")) / "llvm" / "bin" / "llvm-objdump"
PASSES = {"v_mfma_f32_32x32x2_f32": 16, "v_mfma_f32_16x16x4_f32": 8, "v_mfma_f32_16x16x32_bf16": 4, "v_mfma_f32_16x16x32_f16": 4, "v_mfma_f32_32x32x16_bf16": 8,
          "v_mfma_f32_32x32x16_f16": 8, "v_mfma_f32_16x16x128_f8f6f4": 8, "v_mfma_scale_f32_16x16x128_f8f6f4": 8}
OPERAND_STATES, SCALAR_STATES = 2, 5
VECTOR = re.compile(r"\b([av])(?:\[(\d+):(\d+)\]|(\d+))(?![\w\[])")
SCALAR = re.compile(r"\b(s)(?:\[(\d+):(\d+)\]|(\d+))(?![\w\[])")
LINE = re.compile(r"^\t(\S+)(?: (.*?))?\s*// ([0-9A-F]+):.*?(?:<(\S+?)(?:\+0x([0-9a-f]+))?>)?$")


def needed(op):
    return PASSES[op] + (2 if op.endswith("_f32") else 4)


def registers(pattern, text):
    found = set()
    for kind, low, high, one in pattern.findall(text):
        found |= {(kind, int(one))} if one else {(kind, i) for i in range(int(low), int(high) + 1)}
    return found


class Kernel:
    """A function's instructions; branches by the number of the instruction that they go to."""

    def __init__(self, name, lines):
        self.name, self.ops, self.args, places, targets = name, [], [], {}, {}
        for op, args, address, symbol, offset in lines:
            places[int(address, 16)] = len(self.ops)
            if op.startswith(("s_cbranch", "s_branch")) and symbol == name:
                targets[len(self.ops)] = int(offset or "0", 16)
            self.ops.append(op)
            self.args.append(args or "")
        start = min(places)
        self.targets = {at: places[start + offset] for at, offset in targets.items()}
        self.sources = {}
        for at, to in self.targets.items():
            self.sources.setdefault(to, []).append(at)

    def result(self, at):
        return registers(VECTOR, self.args[at].split(",")[0])

    def touched(self, at):
        op = self.ops[at]
        return registers(VECTOR, self.args[at]) if op.startswith(("v_", "ds_", "global_", "buffer_", "flat_", "scratch_")) else set()

    def early_readers(self):
        """(matrix instruction, what touches its result, wait states there) wherever those are too few."""
        found = []
        for first, op in enumerate(self.ops):
            if not op.startswith("v_mfma"):
                continue
            need, seen = needed(op), {}
            ways = [(0, first + 1, frozenset(self.result(first)), PASSES[op] - 1, True)]      # states, place, registers, when the matrix core is free, lanes on
            while ways:
                states, at, live, free, lanes = heapq.heappop(ways)
                if states >= need or at >= len(self.ops) or any(s <= states and live <= l and f <= free and on >= lanes for s, l, f, on in seen.get(at, ())):
                    continue
                seen.setdefault(at, []).append((states, live, free, lanes))
                op, args, states_of = self.ops[at], self.args[at], 1
                if op == "s_endpgm":
                    continue
                if op.startswith("v_mfma"):
                    _, a, b, *_ = args.split(",")
                    if lanes and registers(VECTOR, a + "," + b) & live:
                        found.append((first, at, states))
                    start = max(states, free)
                    if live - self.result(at):
                        heapq.heappush(ways, (start + 1, at + 1, live - self.result(at), start + PASSES[op], lanes))
                    continue
                if lanes and self.touched(at) & live:
                    found.append((first, at, states))
                if op == "s_nop":
                    states_of = int(args, 0) + 1
                if op.startswith("s_") and (args.startswith("exec") or "saveexec" in op):
                    lanes = True
                if at in self.targets:      # a wavefront that goes there without lanes reads nothing until it has some again
                    heapq.heappush(ways, (states + 1, self.targets[at], live, free, lanes and op != "s_cbranch_execz"))
                if op != "s_branch":
                    heapq.heappush(ways, (states + states_of, at + 1, live, free, lanes))
        return found

    def written_late(self, pattern, states_needed, takes, taken):
        """(vector instruction, instruction that ``takes`` a register it writes, wait states between them) wherever those are too few."""
        found = []
        for last, op in enumerate(self.ops):
            registers_taken = registers(pattern, taken(self.args[last])) if takes(op) else ()
            ways, seen = [(0, last, frozenset(registers_taken))], set()
            while ways:
                states, at, live = ways.pop()
                if states >= states_needed or not live or (states, at, live) in seen:
                    continue
                seen.add((states, at, live))
                ways += [(states + 1, source, live) for source in self.sources.get(at, ())]
                at -= 1
                if at < 0 or self.ops[at] in ("s_branch", "s_endpgm"):
                    continue
                op, args = self.ops[at], self.args[at]
                writes = op.startswith(("v_", "s_")) and not op.startswith(("s_cmp", "s_cbranch", "s_waitcnt", "s_nop", "s_barrier"))
                written = registers(pattern, args.split(",")[0]) if writes else set()
                if op.startswith("v_") and not op.startswith("v_mfma") and written & live:
                    found.append((at, last, states))
                ways.append((states + (int(args, 0) + 1 if op == "s_nop" else 1), at, live - written))
        return found

    def early_requests(self):
        return self.written_late(SCALAR, SCALAR_STATES, lambda op: op.startswith(("buffer_", "global_", "flat_")), lambda args: args)

    def early_products(self):
        return self.written_late(VECTOR, OPERAND_STATES, lambda op: op.startswith("v_mfma"), lambda args: args.partition(",")[2])


def kernels(path):
    name, lines = None, []
    text = subprocess.run([str(OBJDUMP), "-d", "--no-show-raw-insn", path], stdout=subprocess.PIPE, text=True, check=True).stdout
    for line in text.splitlines():
        if line.endswith(">:"):
            if lines:
                yield Kernel(name, lines)
            name, lines = line.split("<")[1][:-2], []
        elif line.startswith("\t"):
            match = LINE.match(line)
            if match:
                lines.append(match.groups())
    if lines:
        yield Kernel(name, lines)


def faults(path):
    found, matrix = [], 0
    for kernel in kernels(path):
        matrix += sum(op.startswith("v_mfma") for op in kernel.ops)
        for first, at, states in kernel.early_readers() + kernel.early_requests() + kernel.early_products():
            found.append(f"{kernel.name}: {kernel.ops[first]} {kernel.args[first]} -> {kernel.ops[at]} {kernel.args[at]} after {states}")
    return found, matrix


def code_objects(library, folder):
    """The library's parts for the GPU, one for each source."""
    data, magic, at, paths = library.read_bytes(), b"__CLANG_OFFLOAD_BUNDLE__", -1, []
    while (at := data.find(magic, at + 1)) >= 0:
        (count,), entry = struct.unpack_from("<Q", data, at + len(magic)), at + len(magic) + 8
        for _ in range(count):
            offset, size, length = struct.unpack_from("<QQQ", data, entry)
            if size and b"amdgcn" in data[entry + 24:entry + 24 + length]:
                paths.append(folder / f"{len(paths)}.co")
                paths[-1].write_bytes(data[at + offset:at + offset + size])
            entry += 24 + length
    return [str(path) for path in paths]


@pytest.mark.skipif(not OBJDUMP.exists(), reason="no llvm-objdump")
def test_results_are_waited_for(tmp_path):
    paths = code_objects(LIBRARY, tmp_path)
    assert paths
    with ProcessPoolExecutor(min(8, os.cpu_count())) as pool:
        reports = list(pool.map(faults, paths))
    assert sum(matrix for _, matrix in reports) > 1000
    found = [fault for report, _ in reports for fault in report]
    assert not found, f"{len(found)} places, among them " + "; ".join(found[:6])


def made(*lines):
    text = [f"\t{line.ljust(50)} // {4 * i:012X}: 00000000" + (f" <f+0x{4 * to:x}>" if to is not None else "") for i, (line, to) in enumerate(lines)]
    return Kernel("f", [LINE.match(line).groups() for line in text])


def test_the_reading_of_ways():
    product, reader = ("v_mfma_f32_32x32x2_f32 a[0:15], v1, v2, a[0:15]", None), ("v_accvgpr_read_b32 v3, a15", None)
    assert made(product, ("s_nop 15", None), ("s_nop 1", None), reader).early_readers() == []
    assert made(product, ("s_nop 15", None), ("s_nop 0", None), reader).early_readers() == [(0, 3, 17)]
    # the way that leaves out instruction 2 is the shorter one
    assert made(product, ("s_cbranch_scc1 1", 3), ("s_nop 9", None), ("s_nop 9", None), reader).early_readers() == [(0, 4, 11)]
    assert made(product, ("v_mfma_f32_32x32x2_f32 a[16:31], v1, v2, a[16:31]", None), ("s_nop 1", None), reader).early_readers() == []
    assert made(product, ("v_mfma_f32_32x32x2_f32 a[0:15], v1, v2, a[0:15]", None), ("s_nop 1", None), reader).early_readers() == [(1, 3, 2)]
    operand = ("v_perm_b32 v1, v3, v4, v5", None)
    assert made(operand, product).early_products() == [(0, 1, 0)] and made(operand, ("s_nop 0", None), product).early_products() == [(0, 2, 1)]
    assert made(operand, ("s_nop 1", None), product).early_products() == [] == made(product, product).early_products()
    request = ("buffer_load_dwordx4 v1, s[4:7], s8 offen lds", None)
    assert made(("v_readfirstlane_b32 s8, v1", None), ("s_nop 2", None), request).early_requests() == [(0, 2, 3)]
    assert made(("v_readfirstlane_b32 s8, v1", None), ("s_nop 4", None), request).early_requests() == []
    assert made(("v_readfirstlane_b32 s8, v1", None), ("s_mov_b32 s8, s9", None), request).early_requests() == []

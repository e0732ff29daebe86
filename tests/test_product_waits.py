"""Wait states around matrix products in the device code of the sources that write some of them in assembly, where the compiler counts none.

Read from the compiler's own listing of the sources, along every path that leads to an instruction:
* a vector instruction's result needs two wait states before a product reads it;
* a product's result needs its passes and four more before anything but a product reads or overwrites it, or a product reads it other than as the whole
  of its accumulator.
A pair of instructions that the compiler chose both of is its own business; here one of the two at least is in assembly."""
import os
import re
import subprocess

import pytest

from pypto_amd import build

PASSES = {"v_mfma_f32_32x32x16_bf16": 8, "v_mfma_f32_32x32x16_f16": 8, "v_mfma_f32_16x16x32_bf16": 4, "v_mfma_f32_16x16x32_f16": 4}
BEFORE = 2


def registers(operand):
    m = re.match(r"-?\|?([va])(?:\[(\d+):(\d+)\]|(\d+)\b)", operand)
    if not m:
        return frozenset()
    lo, hi = (int(m[2]), int(m[3])) if m[2] else (int(m[4]), int(m[4]))
    return frozenset((m[1], i) for i in range(lo, hi + 1))


class Instruction:
    def __init__(self, line, number, assembly):
        self.number, self.assembly, self.text = number, assembly, line
        self.op, _, rest = line.partition(" ")
        self.operands = [x.strip() for x in rest.split(",")]
        self.product = self.op.startswith(("v_mfma", "v_smfmac"))
        self.waits = int(self.operands[0], 0) + 1 if self.op == "s_nop" else 1
        sets = [registers(x) for x in self.operands]
        both = self.op.startswith(("v_permlane16_swap", "v_permlane32_swap", "v_swap"))
        stores = self.op.startswith(("ds_write", "ds_store", "global_store", "buffer_store", "scratch_store"))
        self.writes = frozenset() if stores else (sets[0] | sets[1] if both else (sets[0] if sets else frozenset()))
        self.touches = frozenset().union(*sets)
        self.accumulator = sets[3] if self.product else None
        self.factors = sets[1] | sets[2] if self.product else None
        self.vector = self.op.startswith("v_") and not self.product


def read(listing):
    """Functions of a listing: instructions and, of each, those that may come before it."""
    code, labels, before, assembly, jumps, open_end = [], {}, [], False, [], None
    for number, line in enumerate(listing.splitlines(), 1):
        if "ASMSTART" in line or "ASMEND" in line:
            assembly = "ASMSTART" in line
            continue
        text = re.sub(r"\s+", " ", line.split(";")[0].split("//")[0]).strip()
        if re.match(r"^[.\w$]+:", text):
            name = text.split(":")[0]
            labels[name] = len(code)
            if not name.startswith("."):
                open_end = None                            # a function begins
            continue
        if not text or text.startswith("."):
            continue
        x = Instruction(text, number, assembly)
        before.append(set() if open_end is None else {open_end})
        code.append(x)
        open_end = len(code) - 1
        if x.op.startswith(("s_cbranch", "s_branch")):
            jumps.append((len(code) - 1, x.operands[-1]))
        if x.op in ("s_branch", "s_endpgm", "s_setpc_b64"):
            open_end = None
    for at, label in jumps:
        if labels[label] < len(code):
            before[labels[label]].add(at)
    return code, before


def earlier(code, before, at, states):
    """Instructions fewer than `states` wait states in front of instruction `at`, on any path."""
    seen, todo = {}, [(p, 0) for p in before[at]]
    while todo:
        i, waited = todo.pop()
        if waited >= states or seen.get(i, states) <= waited:
            continue
        seen[i] = waited
        todo += [(p, waited + code[i].waits) for p in before[i]]
    return {i: code[i] for i in seen}.values()


def too_close(listing):
    code, before = read(listing)
    found, products = [], 0
    longest = max(PASSES.values()) + 4
    for at, x in enumerate(code):
        products += x.product and x.assembly
        if not x.touches:
            continue
        if x.product:
            for y in earlier(code, before, at, BEFORE):
                if y.vector and (x.assembly or y.assembly) and y.writes & (x.factors | x.accumulator):
                    found.append((y, x))
        for y in earlier(code, before, at, longest):
            if not y.product or not (x.assembly or y.assembly) or y not in earlier(code, before, at, PASSES[y.op] + 4):
                continue
            if (x.factors & y.writes) or (x.accumulator & y.writes and x.accumulator != y.writes) if x.product else x.touches & y.writes:
                found.append((y, x))
    return [f"{y.number}: {y.text}  ->  {x.number}: {x.text}" for y, x in found], products


PRODUCT = "v_mfma_f32_32x32x16_bf16 v[0:15], v[20:23], v[24:27], {}\n"


@pytest.mark.parametrize("listing,bad", [
    ("f:\nv_mov_b32_e32 v20, v1\n#\n" + PRODUCT.format("v[0:15]") + "$\n", 1),
    ("f:\nv_mov_b32_e32 v20, v1\ns_nop 1\n#\n" + PRODUCT.format("0") + "$\n", 0),
    ("f:\nv_mov_b32_e32 v20, v1\nv_mov_b32_e32 v29, v1\n#\n" + PRODUCT.format("0") + "$\n", 1),
    ("f:\nv_mov_b32_e32 v28, v1\n#\n" + PRODUCT.format("0") + "$\n", 0),
    ("f:\n#\nv_mov_b32 v27, v1\n$\n" + PRODUCT.format("0"), 1),                                             # only the writer in assembly
    ("f:\nv_mov_b32_e32 v27, v1\n" + PRODUCT.format("0"), 0),                                               # neither
    ("f:\n#\n" + PRODUCT.format("0") + "$\n#\n" + PRODUCT.format("v[0:15]") + "$\n", 0),
    ("f:\n#\n" + PRODUCT.format("0") + "$\ns_nop 10\nv_add_f32_e32 v30, v15, v31\n", 1),
    ("f:\n#\n" + PRODUCT.format("0") + "$\ns_nop 11\nv_add_f32_e32 v30, v15, v31\n", 0),
    ("f:\n#\n" + PRODUCT.format("0") + "$\nds_write_b32 v30, v15\n", 1),
    ("f:\n#\n" + PRODUCT.format("0") + "$\nv_mov_b32_e32 v3, v40\n", 1),
    ("f:\n.L1:\n#\n" + PRODUCT.format("0") + "$\ns_nop 15\nv_mov_b32_e32 v22, v1\ns_cbranch_scc1 .L1\n", 1),   # round the loop, behind a branch
    ("f:\n.L1:\n#\n" + PRODUCT.format("0") + "$\ns_nop 15\nv_mov_b32_e32 v22, v1\ns_nop 0\ns_cbranch_scc1 .L1\n", 0),
    ("f:\nv_mov_b32_e32 v20, v1\ns_endpgm\ng:\n#\n" + PRODUCT.format("0") + "$\n", 0),
])
def test_the_rules(listing, bad):
    found, _ = too_close(listing.replace("#", ";;#ASMSTART").replace("$", ";;#ASMEND"))
    assert len(found) == bad, found


@pytest.mark.parametrize("source", ["latent_wide.hip", "sfa_kernels.hip"])
def test_products_in_assembly(source, tmp_path):
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    if not os.path.exists(hipcc):
        pytest.skip("no compiler")
    flags = [f for f in build.HIPCC_FLAGS if f not in ("-shared", "-fPIC")]
    out = tmp_path / "listing.s"
    subprocess.run([hipcc, *flags, "-w", "-x", "hip", "-I" + build.INCLUDE, "-I" + build.CSRC, "-S", "--cuda-device-only", os.path.join(build.CSRC, source), "-o", str(out)],
                   check=True, stderr=subprocess.DEVNULL)
    found, products = too_close(out.read_text())
    assert products > 0 and not found, "\n".join(found[:20])


def test_no_other_source_has_products_in_assembly():
    pattern = re.compile(r"asm[^;]*?\"[^;]*v_mfma", re.S)
    having = {f for f in os.listdir(build.CSRC) if pattern.search(open(os.path.join(build.CSRC, f)).read())}
    assert having == {"latent_wide.hip", "sfa_kernels.hip"}

"""What the compiler does not check in the kernels of include/bof_f8.h, read from the built library's own gfx950 code:

The matrix instructions of the large tiles and the loads to LDS are inline assembly, around which the compiler puts no wait
states.  On every path through a kernel
  * no vector instruction writes an operand, an accumulator or a scale of a matrix instruction in the two wait states in front
    of it;
  * nothing but a matrix instruction with the very same accumulator touches an accumulator in the wait states that its
    result takes (11 behind the f8 instructions, 7 behind the bf16 ones);
  * no vector instruction writes a scalar register in the five wait states in front of a load to LDS that addresses with it,
    and M0 is written one wait state or more ahead of the load.
"""
import collections
import glob
import os
import re
import subprocess

import pytest

import bofhip

OBJDUMP = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin", "llvm-objdump")
Ins = collections.namedtuple("Ins", "at op args target")   # address, mnemonic, operands, branch target (offset in the kernel)


def parse(text):
    """{kernel: [Ins]} of llvm-objdump's disassembly."""
    kernels, body = {}, None
    for line in text.splitlines():
        head = re.match(r"([0-9a-f]+) <(.*)>:", line)
        if head:
            body = kernels.setdefault(head.group(2), [])
        elif body is not None and line.startswith("\t") and "//" in line:
            code, _, note = line.partition("//")
            op, _, args = code.strip().partition(" ")
            to = re.search(r"<[^>]*?(?:\+0x([0-9a-f]+))?>", note)
            body.append(Ins(int(re.match(r"\s*([0-9A-F]+):", note).group(1), 16), op,
                            [a.strip() for a in re.split(r",(?![^\[]*\])", args)], int(to.group(1) or "0", 16) if to else None))
    return kernels


def registers(text):
    """{(kind, number)} of the vector, accumulator and scalar registers named in a text."""
    return {(kind, i) for kind, lo, hi, one in re.findall(r"\b([avs])(?:\[(\d+):(\d+)\]|(\d+)\b)", text)
            for i in range(int(lo or one), int(hi or one) + 1)} | ({("m0", 0)} if re.search(r"\bm0\b", text) else set())


def written(ins):
    """Registers a vector instruction writes (matrix instructions aside)."""
    if not ins.op.startswith("v_") or ins.op.startswith(("v_mfma", "v_nop")):
        return set()
    return registers(ins.args[0]) | (registers(ins.args[1]) if ins.op.startswith("v_swap") else set())


def states(ins):
    return int(ins.args[0]) + 1 if ins.op == "s_nop" else 1


class Flow:
    def __init__(self, body):
        self.body, at = body, {i.at: n for n, i in enumerate(body)}
        self.before, self.behind = collections.defaultdict(list), collections.defaultdict(list)
        for n, i in enumerate(body):
            to = [at[body[0].at + i.target]] if i.op.startswith(("s_cbranch", "s_branch")) else []
            if i.op not in ("s_branch", "s_endpgm") and n + 1 < len(body):
                to.append(n + 1)
            for t in to:
                self.behind[n].append(t)
                self.before[t].append(n)

    def within(self, n, limit, back):
        """Every instruction that fewer than `limit` wait states part from instruction n, on any path; send(True) ends the path."""
        step, todo, seen = self.before if back else self.behind, [], set()
        todo += [(p, 0) for p in step[n]]
        while todo:
            p, d = todo.pop()
            if d >= limit or (p, d) in seen:
                continue
            seen.add((p, d))
            if not (yield self.body[p]):
                todo += [(q, d + states(self.body[p])) for q in step[p]]


def each(walk):
    """The walk with paths that never end early."""
    try:
        i = next(walk)
        while True:
            yield i
            i = walk.send(False)
    except StopIteration:
        return


def faults(body):
    """Descriptions of all that the compiler may have put too close to a matrix instruction or to a load to LDS."""
    flow, found = Flow(body), []
    for n, i in enumerate(body):
        def wrong(what, other):
            found.append(f"{i.at:x}: {i.op} {', '.join(i.args)}: {what} by {other.op} {', '.join(other.args)}")
        if i.op.startswith("v_mfma"):
            reads, acc = registers(" ".join(i.args[1:])), registers(i.args[0])
            for p in each(flow.within(n, 2, back=True)):
                if written(p) & (reads | acc):
                    wrong("an operand is written just before", p)
            walk = flow.within(n, 11 if "f8f6f4" in i.op else 7, back=False)
            try:
                p = next(walk)
                while True:
                    same = p.op.startswith("v_mfma") and registers(p.args[0]) == acc and registers(p.args[3]) == acc
                    if same and registers(" ".join(p.args[1:3])) & acc or not same and registers(" ".join(p.args)) & acc:
                        wrong("the result is touched too early", p)
                    p = walk.send(same)
            except StopIteration:
                pass
        elif i.op.startswith("global_load_lds"):
            base = {r for r in registers(" ".join(i.args)) if r[0] == "s"}
            for p in each(flow.within(n, 5, back=True)):
                if p.op.startswith("v_") and registers(p.args[0]) & base:
                    wrong("its address is written just before", p)
            for p in each(flow.within(n, 1, back=True)):
                if ("m0", 0) in registers(p.args[0]):
                    wrong("M0 is written just before", p)
    return found


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    if not os.path.exists(OBJDUMP):
        pytest.skip("no llvm-objdump")
    bofhip.lib()
    where = tmp_path_factory.mktemp("code")
    os.symlink(bofhip.LIB_PATH, where / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=where, check=True, capture_output=True)
    found = {}
    for path in glob.glob(str(where / "*gfx950")):
        if b"f8_ring_kernel" in open(path, "rb").read():
            found.update(parse(subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", path], check=True, capture_output=True, text=True).stdout))
    return found


def test_matrix_instructions_and_loads_to_lds_have_their_wait_states(kernels):
    products = {k: body for k, body in kernels.items() if re.search("f8_(tile|ring|wide|rows)", k)}
    assert len(products) >= 4 * 16 and sum(i.op.startswith("v_mfma") for b in products.values() for i in b) > 4000
    bad = {k: f for k, f in ((k, faults(body)) for k, body in products.items()) if f}
    assert not bad, "\n".join(f"{k}: {len(f)} places, the first: {f[0]}" for k, f in bad.items())


def test_the_product_loads_memory_as_memory(kernels):
    """A load through an address of any kind (flat) also counts as one of LDS: the wait for fragments in front of a barrier would
    wait for the rows that are to arrive two steps later."""
    for name, body in kernels.items():
        if "f8_" in name:
            assert not [i.op for i in body if i.op.startswith("flat_")], name


MFMA = "v_mfma_scale_f32_16x16x128_f8f6f4 a[0:3], v[2:9], v[10:17], a[0:3], v18, v19 op_sel_hi:[0,0,0]"


@pytest.mark.parametrize("code,clean", [
    (["v_and_b32_e32 v19, 0xff, v19", MFMA], False),
    (["v_and_b32_e32 v19, 0xff, v19", "s_nop 0", MFMA], False),
    (["v_and_b32_e32 v19, 0xff, v19", "s_nop 1", MFMA], True),
    (["v_accvgpr_read_b32 v9, a95", "s_waitcnt vmcnt(0)", MFMA], False),
    (["v_accvgpr_write_b32 a3, v1", MFMA], False),
    (["v_and_b32_e32 v20, 0xff, v19", MFMA], True),
    (["ds_read_b128 v[2:5], v40", "s_waitcnt lgkmcnt(0)", MFMA], True),
    ([MFMA, MFMA, MFMA], True),
    ([MFMA, "s_nop 7", "v_accvgpr_read_b32 v40, a2"], False),
    ([MFMA, "s_nop 15", "v_accvgpr_read_b32 v40, a2"], True),
    ([MFMA, "v_mov_b32_e32 v40, v2"], True),
    ([MFMA, MFMA.replace("a[0:3]", "a[2:5]")], False),
    ([MFMA, "ds_write_b128 v1, a[0:3]"], False),
    (["v_readfirstlane_b32 s4, v0", "s_mov_b32 m0, s9", "s_nop 0", "global_load_lds_dwordx4 v1, s[4:5]"], False),
    (["v_readfirstlane_b32 s4, v0", "s_mov_b32 m0, s9", "s_nop 3", "global_load_lds_dwordx4 v1, s[4:5]"], True),
    (["s_mov_b32 m0, s9", "global_load_lds_dwordx4 v1, s[4:5]"], False),
])
def test_the_reader_sees_what_it_is_to_see(code, clean):
    text = "0000000000000100 <kernel>:\n" + "".join(f"\t{c}  // {256 + 8 * n:012X}: 00000000\n" for n, c in enumerate(code + ["s_endpgm"]))
    assert (not faults(parse(text)["kernel"])) == clean


def test_the_reader_follows_loops():
    """A write at the end of a loop, its matrix instruction at the loop's head."""
    code = [MFMA, "s_nop 15", "v_and_b32_e32 v18, 0xff, v18", "s_cbranch_scc1 65532", "s_endpgm"]
    notes = ["", "", "", " <kernel+0x0>", ""]
    text = "0000000000000100 <kernel>:\n" + "".join(f"\t{c}  // {256 + 8 * n:012X}: 00000000{notes[n]}\n" for n, c in enumerate(code))
    found = faults(parse(text)["kernel"])
    assert len(found) == 1 and "v_and_b32_e32" in found[0]

"""The machine code of the built library (CPU; compiled here from csrc/): no register of a whole wave is spilled, reloaded or copied
under the lane mask of a branch.

Where lanes that have taken different ways meet again, the code widens the lane mask (`s_or_b64 exec, exec, ..`).  A spill that
the register allocator puts in front of that instruction stores the lanes of one way only -- none, behind a loop that every lane has
left -- and the reload finds what the slot held before.  k_backtrace once lost the address of the tuples it moves in this way: a call
with paths that change state at nearly every frame ended with an illegal address."""
import os
import re
import struct
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "bournemouth-forced-aligner_amd", "libbfa_hip.so")
OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
# what the register allocator inserts: accesses to spill slots, copies of whole registers; and what may stand between them
SPILL = re.compile(r"\tscratch_(?:load|store)_")
COPY = re.compile(r"\tv_mov_b32_e32 v\d+, v\d+\b|\tv_mov_b64_e32 v\[\d+:\d+\], v\[|\tv_accvgpr_")
BETWEEN = re.compile(r"\t(?:v_readlane_b32|v_writelane_b32|s_nop|s_waitcnt)\b")
RESTORE = re.compile(r"\n\ts_or_b64 exec, exec,")
HEAD = re.compile(r"(?:[0-9a-f]+ )?<\w+>:")


def masked_spills(text):
    """[(function, instructions)] of the exec restores with a spill right in front of them, or with nothing but copies between them and
    the head of their block"""
    found = []
    for m in RESTORE.finditer(text):
        seen, spills, at_head = [], 0, False
        for line in reversed(text[max(0, m.start() - 4000):m.start()].split("\n")[1:]):
            if HEAD.match(line):
                at_head = True
                break
            if SPILL.match(line):
                spills += 1
            elif not (COPY.match(line) or BETWEEN.match(line)):
                break
            seen.append(line.split("//")[0].strip())
        if spills or (at_head and any(COPY.match("\t" + s) for s in seen)):
            name = re.findall(r"<(?!L\d+>)(\w+)>:", text[:m.start()])
            found.append((name[-1] if name else "?", seen[::-1]))
    return found


def code_objects(path):
    """the gfx950 ELF images in the library's offload bundles"""
    blob, magic, at, out = open(path, "rb").read(), b"__CLANG_OFFLOAD_BUNDLE__", 0, []
    while (at := blob.find(magic, at)) >= 0:
        n, q = struct.unpack_from("<Q", blob, at + 24)[0], at + 32
        for _ in range(n):
            off, size, length = struct.unpack_from("<QQQ", blob, q)
            if b"gfx950" in blob[q + 24:q + 24 + length] and size:
                out.append(blob[at + off:at + off + size])
            q += 24 + length
        at += len(magic)
    return out


def test_the_check_sees_a_spill_under_a_narrow_mask():
    join = "\n<k>:\n<L4>:\n{}\ts_or_b64 exec, exec, s[6:7]                                // 0: 0\n"
    assert masked_spills(join.format("")) == []
    assert masked_spills(join.format("\tv_add_u32_e32 v1, v2, v3    // 0: 0\n")) == []  # (the work of the branch itself)
    assert masked_spills(join.format("\tscratch_store_dwordx2 off, v[120:121], off offset:16    // 0: 0\n")) == [
        ("k", ["scratch_store_dwordx2 off, v[120:121], off offset:16"])]
    assert masked_spills(join.format("\tv_mov_b32_e32 v7, v9    // 0: 0\n\ts_nop 1    // 0: 0\n")) == [
        ("k", ["v_mov_b32_e32 v7, v9", "s_nop 1"])]


PACKED = re.compile(r"\bv_pk_(?:add|mul|fma)_f32\b")


@pytest.fixture(scope="module")
def library(tmp_path_factory):
    """what stands in the machine code of the built library: [(spills under a narrow mask, packed float32 instructions)] per unit"""
    if not os.path.exists(OBJDUMP):
        pytest.skip("llvm-objdump is not there")
    if not os.path.exists(LIB):
        import __graft_entry__
        __graft_entry__.build()
    tmp_path = tmp_path_factory.mktemp("code")

    def scan(item):
        k, image = item
        f = tmp_path / f"{k}.co"
        f.write_bytes(image)
        text = subprocess.run([OBJDUMP, "-d", "--symbolize-operands", str(f)], capture_output=True, text=True, check=True).stdout
        assert "s_endpgm" in text
        return masked_spills(text), PACKED.findall(text)

    images = code_objects(LIB)
    assert len(images) >= 20
    with ThreadPoolExecutor(4) as pool:
        return list(pool.map(scan, enumerate(images)))


def test_no_spill_under_a_narrow_lane_mask(library):
    found = [x for spills, _ in library for x in spills]
    assert not found, found


def test_no_packed_float32_instructions(library):
    """Some forms of them have given wrong results on this hardware: neither the compiler (a flag) nor inline asm makes them."""
    assert not any(packed for _, packed in library)
    for top in ("bournemouth-forced-aligner_amd/csrc", "tools"):
        for folder, _, names in os.walk(os.path.join(ROOT, top)):
            for name in names:
                if name.endswith((".hip", ".inc", ".hpp", ".cpp")):
                    code = re.sub(r"//.*", "", open(os.path.join(folder, name), errors="replace").read())
                    assert not PACKED.search(code), os.path.join(folder, name)


def test_no_vector_instruction_in_inline_asm_reads_a_scalar_register():
    """The compiler keeps its own vector instructions apart from a v_readlane that has just brought a spilled scalar register back; it
    does not look into inline asm."""
    src = os.path.join(ROOT, "bournemouth-forced-aligner_amd", "csrc")
    for name in sorted(os.listdir(src)):
        if not name.endswith((".hip", ".inc", ".hpp", ".cpp")):
            continue
        for statement in re.findall(r"\basm\b(?:\s+volatile)?\s*\((.*?)\);", open(os.path.join(src, name)).read(), flags=re.S):
            code, _, operands = statement.partition(":")
            if re.search(r'"\s*v_|\\tv_', code):
                assert not re.search(r'"\+?s"\s*\(', operands), f"{name}: {statement[:200]}"

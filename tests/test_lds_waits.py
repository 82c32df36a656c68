"""What the built library's own machine code does at its workgroup barriers (no GPU).

Several kernels refill a slot of LDS by direct copies from memory that are requested right behind a barrier, while other wavefronts
have read that slot before it.  The copies are outside the compiler's memory model, and a barrier alone does not wait for a
wavefront's outstanding LDS reads: a wavefront that meets the barrier with reads in flight may have them overtaken by a copy.  So no
wavefront may meet a barrier with LDS accesses outstanding, whatever path led to it."""
import os
import re
import struct
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

from intel_gaudi3_software_amd import abi

OBJDUMP = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin", "llvm-objdump")
MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"


def code_objects(path):
    """The gfx950 code objects of a shared library, in the order in which they were linked."""
    with open(path, "rb") as f:
        data = f.read()
    found, at = [], data.find(MAGIC)
    while at >= 0:
        entries, p = struct.unpack_from("<Q", data, at + len(MAGIC))[0], at + len(MAGIC) + 8
        for _ in range(entries):
            offset, size, length = struct.unpack_from("<QQQ", data, p)
            name = data[p + 24:p + 24 + length]
            p += 24 + length
            if name.endswith(b"gfx950") and size:
                found.append(data[at + offset:at + offset + size])
        at = data.find(MAGIC, at + 1)
    return found


HEAD = re.compile(r"^([0-9a-f]+) <(.*)>:$")
LINE = re.compile(r"^\t(\S+)(.*?)// ([0-9A-F]+):.*?(?:<.*\+0x([0-9a-f]+)>)?$")
LGKM = re.compile(r"lgkmcnt\((\d+)\)")
ENDS = ("s_branch", "s_endpgm", "s_setpc_b64", "always")
ZERO = re.compile(r"^\ts_mov_b64 (s\[\d+:\d+\]), 0 +// ([0-9A-F]+):")


def functions(text):
    """(name, [(address, mnemonic, operands, branch target)]) of every function, only what the analysis looks at.  A condition that is set
    to zero right in front of the branch on it (how the compiler ends the first of two alternatives, the second of which others
    enter at the branch) is a branch that is always taken by whoever comes past the setting: "always"."""
    name, start, lines, before = None, 0, [], ("", "")
    for line in text.splitlines():
        if not line.startswith("\t"):
            m = HEAD.match(line)
            if m:
                if name:
                    yield name, lines
                name, start, lines, before = m.group(2), int(m.group(1), 16), [], ("", "")
            continue
        if line.startswith(("\tds_", "\ts_waitcnt", "\ts_barrier", "\ts_cbranch", "\ts_branch", "\ts_endpgm", "\ts_setpc", "\tglobal_load_lds", "\tbuffer_load")):
            m = LINE.match(line)
            target = start + int(m.group(4), 16) if m.group(4) else start if "branch" in m.group(1) and "// " in line and line.endswith(">") else None
            zero = ZERO.match(before[0])
            if m.group(1) == "s_cbranch_vccz" and zero and before[1].startswith("\ts_and_b64 vcc, exec, %s " % zero.group(1)):
                lines.append((int(zero.group(2), 16), "always", "", target))
            lines.append((int(m.group(3), 16), m.group(1), m.group(2), target))
        before = (before[1], line)
    if name:
        yield name, lines


def outstanding_at_barriers(lines):
    """For every barrier the largest number of LDS accesses a wavefront may have in flight there.  A wait for lgkmcnt(n) leaves at most n
    of them; the count along every path is followed until it no longer grows (up to the counter's 15)."""
    addresses = [l[0] for l in lines]

    def first_at(address):  # index of the first line of interest at or behind an address
        import bisect
        return bisect.bisect_left(addresses, address)

    state, at_barrier, todo = {0: 0}, {}, [0]
    while todo:
        i = todo.pop()
        n = state[i]
        while i < len(lines):
            _, op, operands, target = lines[i]
            if op.startswith("ds_"):
                n = min(n + 1, 15)
            elif op == "s_waitcnt":
                m = LGKM.search(operands)
                if m:
                    n = min(n, int(m.group(1)))
            elif op == "s_barrier":
                at_barrier[i] = max(at_barrier.get(i, 0), n)
            if target is not None:
                j = first_at(target)
                if j < len(lines) and state.get(j, -1) < n:
                    state[j] = n
                    todo.append(j)
            i += 1
            if op in ENDS:
                break
            if i in state or (i < len(lines) and op.startswith("s_cbranch")):
                if state.get(i, -1) >= n:
                    break
                state[i] = n
    return at_barrier


@pytest.fixture(scope="module")
def kernels():
    """name -> (outstanding at its barriers, whether it requests copies to LDS) of every function of the library that has a barrier."""
    if not os.path.exists(abi.LIB_PATH):
        pytest.skip("libmme_hip.so has not been built (python -m intel_gaudi3_software_amd.build)")
    if not os.path.exists(OBJDUMP):
        pytest.skip("no llvm-objdump")

    def listing(code):
        r = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", "-"], input=code, stdout=subprocess.PIPE, check=True)
        return r.stdout.decode(errors="replace")

    found = {}
    with ThreadPoolExecutor(4) as pool:
        for text in pool.map(listing, code_objects(abi.LIB_PATH)):
            for name, lines in functions(text):
                barriers = outstanding_at_barriers(lines)
                if barriers:
                    found[name] = (list(barriers.values()), any("lds" in l[1] for l in lines))
    return found


def test_the_analysis_itself():
    listing = ("0000000000001000 <k>:\n"
               "\tds_read_b128 v[0:3], v4                                    // 000000001000: D9FE0000\n"
               "\ts_waitcnt vmcnt(8)                                         // 000000001008: BF8C0F78\n"
               "\ts_barrier                                                  // 00000000100C: BF8A0000\n"
               "\ts_waitcnt lgkmcnt(0)                                       // 000000001010: BF8CC07F\n"
               "\ts_barrier                                                  // 000000001014: BF8A0000\n"
               "\tds_read_b128 v[0:3], v4                                    // 000000001018: D9FE0000\n"
               "\ts_cbranch_scc1 65534                                       // 000000001020: BF85FFFE <k+0x14>\n"
               "\ts_endpgm                                                   // 000000001024: BF810000\n")
    (name, lines), = functions(listing)
    assert name == "k" and list(outstanding_at_barriers(lines).values()) == [1, 15]
    fixed = listing.replace("s_waitcnt vmcnt(8) ", "s_waitcnt vmcnt(8) lgkmcnt(0) ").replace("\ts_cbranch_scc1", "\ts_waitcnt lgkmcnt(0) // 00000000101C:\n\ts_cbranch_scc1")
    (_, lines), = functions(fixed)
    assert list(outstanding_at_barriers(lines).values()) == [0, 0]
    # two alternatives: the end of the first never enters the second, which is entered at the branch
    listing = ("0000000000002000 <k>:\n"
               "\ts_cbranch_scc0 9                                           // 000000002000: BF840009 <k+0x18>\n"
               "\tds_write_b128 v4, v[0:3]                                   // 000000002004: D9BE0000\n"
               "\ts_mov_b64 s[6:7], 0                                        // 000000002010: BE860180\n"
               "\ts_and_b64 vcc, exec, s[6:7]                                // 000000002018: 86EA067E\n"
               "\ts_cbranch_vccz 3                                           // 00000000201C: BF860003 <k+0x28>\n"
               "\ts_barrier                                                  // 000000002020: BF8A0000\n"
               "\ts_endpgm                                                   // 000000002028: BF810000\n")
    (_, lines), = functions(listing)
    assert list(outstanding_at_barriers(lines).values()) == [0]
    (_, lines), = functions(listing.replace("s_mov_b64 s[6:7], 0 ", "s_mov_b64 s[6:7], -1"))
    assert list(outstanding_at_barriers(lines).values()) == [1]


def test_scaled_product_has_no_lds_access_in_flight_at_a_barrier(kernels):
    mine = {n: k for n, k in kernels.items() if "scaled_gemm" in n}
    assert len(mine) > 60 and any("large" in n for n in mine) and all(k[1] for n, k in mine.items() if "large" in n)
    assert not {n: k[0] for n, k in mine.items() if max(k[0])}


def test_no_kernel_has_an_lds_access_in_flight_at_a_barrier(kernels):
    assert sum(k[1] for k in kernels.values()) > 150  # (kernels that request copies to LDS)
    assert not {n: k[0] for n, k in kernels.items() if max(k[0])}

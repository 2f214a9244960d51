"""Copies from global memory to LDS are asynchronous, and a barrier does not wait for them: a wave that passes it with copies under way publishes rows that
are not there yet.  Every kernel of the built library that makes such copies is followed instruction by instruction, along all branches: no barrier, and
no end of a wave, is reached with a copy that no wait on the vector-memory counter has covered, and no barrier with an access to LDS that no wait
on its counter has covered."""
import os
import re
import shutil
import subprocess

import pytest

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
COPY = re.compile(r"^(global_load_lds_|buffer_load_\S+ .*\blds\b)")
VECTOR_MEMORY = re.compile(r"^(global|buffer|scratch|flat|tbuffer|image)_(?!wbl2|inv)")
LDS = re.compile(r"^ds_(?!bpermute|permute|swizzle)")
TARGET = re.compile(r"<([^<>]+?)(?:\+0x([0-9a-f]+))?>\s*$")


def kernels(listing):
    """(name, [(address, instruction)]) of the functions of a disassembly."""
    name, code = None, []
    for line in listing:
        if line.endswith(">:\n"):
            if name:
                yield name, code
            name, code = line.split("<", 1)[1][:-3], []
        elif line.startswith("\t") and "//" in line:
            text, _, note = line.partition("//")
            code.append((int(note.split(":")[0], 16), text.strip(), note))
    if name:
        yield name, code


def uncovered(code, first=COPY, later=VECTOR_MEMORY, counter="vmcnt", places=("s_barrier", "s_endpgm")):
    """Places (address, instruction) that a wave may reach with a copy to LDS that is not waited for.  Followed for every instruction: the smallest
    number of vector-memory operations issued since the youngest copy that may be under way, None where there is none; operations end in order, so
    vmcnt(n) covers it if that number is at least n.  Other operations and counters likewise; without `later` only a wait for 0 counts."""
    counter = re.compile(counter + r"\((\d+)\)")
    at = {a: i for i, (a, _, _) in enumerate(code)}
    state, todo, bad = {0: None}, [0], set()
    while todo:
        i = todo.pop()
        k = state[i]
        while True:
            address, text, note = code[i]
            op = text.split(None, 1)[0]
            if first.match(text):
                k = 0
            elif later and later.match(op) and k is not None:
                k += 1
            elif op == "s_waitcnt":
                wait = counter.search(text)
                if wait and k is not None and k >= int(wait.group(1)):
                    k = None
            elif op in places and k is not None:
                bad.add((address, op))
            assert op not in ("s_setpc_b64", "s_swappc_b64", "s_call_b64"), "calls are not followed"
            follow = [] if op in ("s_endpgm", "s_branch") else [i + 1]
            if op.startswith(("s_branch", "s_cbranch")):
                target = TARGET.search(note)
                follow.append(at[code[0][0] + int(target.group(2) or "0", 16)])
            go_on = None
            for j in follow:
                if j not in state or (k is not None and (state[j] is None or k < state[j])):
                    state[j] = k
                    if go_on is None:
                        go_on = j
                    else:
                        todo.append(j)
            if go_on is None:
                break
            i = go_on
    return sorted(bad)


def program(*lines):
    return [(4 * i, text, note) for i, (text, note) in enumerate(l if isinstance(l, tuple) else (l, "") for l in lines)]


def test_the_check_itself():
    copy, store = "global_load_lds_dwordx4 v[0:1], off", "global_store_dwordx4 v[0:1], v[2:5], off"
    jump = lambda to: ("s_cbranch_scc1 1", f" 0: 0 <kernel+0x{4 * to:x}>")
    assert not uncovered(program(copy, "s_waitcnt vmcnt(0)", "s_barrier", "s_endpgm"))
    assert uncovered(program(copy, "s_waitcnt lgkmcnt(0)", "s_barrier", "s_waitcnt vmcnt(0)", "s_endpgm")) == [(8, "s_barrier")]
    assert not uncovered(program(copy, store, "s_waitcnt vmcnt(1) lgkmcnt(0)", "s_barrier", "s_endpgm"))
    assert uncovered(program(copy, store, "s_waitcnt vmcnt(2)", "s_barrier", "s_waitcnt vmcnt(0)", "s_endpgm")) == [(12, "s_barrier")]
    # copied behind the barrier, waited for on one way back to it only
    assert uncovered(program("s_barrier", copy, jump(4), "s_waitcnt vmcnt(0)", jump(0), "s_waitcnt vmcnt(0)", "s_endpgm")) == [(0, "s_barrier")]
    assert not uncovered(program("s_barrier", copy, "s_waitcnt vmcnt(0)", jump(0), "s_endpgm"))
    assert uncovered(program(copy, "s_endpgm")) == [(4, "s_endpgm")]
    lds = lambda code: uncovered(code, LDS, None, "lgkmcnt", ("s_barrier",))
    assert lds(program("ds_write_b32 v0, v1", "s_load_dword s0, s[2:3], 0x0", "s_waitcnt lgkmcnt(1)", "s_barrier", "s_endpgm")) == [(12, "s_barrier")]
    assert not lds(program("ds_read_b32 v0, v1", "s_waitcnt vmcnt(3) lgkmcnt(0)", "s_barrier", "ds_write_b32 v0, v1", "s_endpgm"))


def test_copies_to_lds_are_waited_for(tmp_path):
    from nemo_amd import _lib
    if not os.path.exists(_lib.LIB_PATH) or not os.path.exists(OBJDUMP):
        pytest.skip("libnemo_hip.so is not built, or there is no disassembler")
    library = shutil.copy(_lib.LIB_PATH, tmp_path / "library.so")          # the device code is written beside it
    subprocess.run([OBJDUMP, "--offloading", library], check=True, stdout=subprocess.DEVNULL)
    copying, found = 0, []
    for part in sorted(tmp_path.glob("library.so.*gfx950*")):
        listing = subprocess.run([OBJDUMP, "-d", part], check=True, stdout=subprocess.PIPE, text=True).stdout
        for name, code in kernels(listing.splitlines(keepends=True)):
            if any(COPY.match(text) for _, text, _ in code):
                copying += 1
                places = uncovered(code) + uncovered(code, LDS, None, "lgkmcnt", ("s_barrier",))
                if places:
                    found.append(f"{name}: {', '.join(f'{op} at {address - code[0][0]:#x}' for address, op in places)}")
    assert copying > 0
    assert not found, f"{len(found)} of {copying} kernels:\n" + "\n".join(found)

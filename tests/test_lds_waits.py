"""Static check of the built kernels: no LDS read of the 8-bit linears or the masked attention is in flight across a
workgroup barrier.  Behind the barrier another wave may refill the stage that the read takes from; only the read's own
wait (``lgkmcnt``) orders the two, and hipcc puts it before the first use, which may come after the barrier."""
import re
import shutil
import subprocess
from pathlib import Path

import pytest

from arbius_amd.ops.build import LIB

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
LINE = re.compile(r"^\s+(\S+)(.*?)//\s*([0-9A-F]{12}):")
TARGET = re.compile(r"<[^>]*?(?:\+0x([0-9a-f]+))?>\s*$")
WAIT = re.compile(r"lgkmcnt\((\d+)\)")
KEPT = (1 << 64) - 1


def functions(listing):
    """name, [(address, opcode, operands, branch target or None)] of every function of a listing."""
    name, base, code = None, 0, []
    for line in listing.splitlines():
        head = re.match(r"^([0-9a-f]{16}) <(.+)>:$", line)
        if head:
            if code:
                yield name, code
            name, base, code = head.group(2), int(head.group(1), 16), []
            continue
        m = LINE.match(line)
        if not m:
            continue
        op, target = m.group(1), None
        if op.startswith(("s_branch", "s_cbranch")):
            t = TARGET.search(line)
            target = base + int(t.group(1) or "0", 16)
        code.append((int(m.group(3), 16), op, m.group(2), target))
    if code:
        yield name, code


def reads_at_barriers(code):
    """Addresses of the barriers that some path reaches with LDS reads in flight.  A state is a bit per outstanding
    LDS / scalar operation, the newest lowest, set for reads; paths that meet are joined bit by bit."""
    at = {c[0]: i for i, c in enumerate(code)}
    state, work, bad = {0: 0}, [0], set()
    while work:
        i = work.pop()
        mask = state[i]
        while True:
            addr, op, rest, target = code[i]
            if op.startswith("ds_") or op.startswith("s_load") or op.startswith("s_buffer_load"):
                mask = (mask << 1 | op.startswith("ds_read")) & KEPT
            elif op == "s_waitcnt":
                w = WAIT.search(rest)
                if w:
                    mask &= (1 << int(w.group(1))) - 1
            elif op == "s_barrier" and mask:
                bad.add(addr)
            nxt = ([] if op in ("s_endpgm", "s_branch", "s_setpc_b64") else [i + 1]) + \
                ([at[target]] if target is not None else [])
            if nxt == [i + 1] and i + 1 not in state:
                i += 1                       # straight on; joins are the only states kept
                if i in joins(code, at):
                    state[i] = mask
                continue
            for j in nxt:
                if j not in state or state[j] | mask != state[j]:
                    state[j] = state.get(j, 0) | mask
                    work.append(j)
            break
    return sorted(bad)


_JOINS = {}


def joins(code, at):
    key = id(code)
    if key not in _JOINS:
        _JOINS.clear()
        _JOINS[key] = {at[c[3]] for c in code if c[3] is not None}
    return _JOINS[key]


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    if not Path(OBJDUMP).exists() or not LIB.exists():
        pytest.skip("no built kernels or no disassembler")
    tmp = tmp_path_factory.mktemp("asm")
    shutil.copy(LIB, tmp / "k.so")
    subprocess.run([OBJDUMP, "--offloading", "k.so"], cwd=tmp, check=True, capture_output=True)
    found = {}
    for f in sorted(tmp.glob("k.so.*amdgcn*")):
        blob = f.read_bytes()
        if b"linear_int8_rows_kernel" in blob or b"masked_attention_kernel" in blob:
            out = subprocess.run([OBJDUMP, "-d", str(f)], check=True, capture_output=True, text=True).stdout
            found.update(functions(out))
    return found


def test_the_check_sees_a_read_across_a_barrier():
    def code(*ops):
        return [(4 * i, o.split()[0], o[len(o.split()[0]):], None) for i, o in enumerate(ops)]
    loop = code("ds_read_b128 v[0:3], v4", "s_barrier", "s_waitcnt lgkmcnt(0)", "s_endpgm")
    assert reads_at_barriers(loop) == [4]
    assert reads_at_barriers(code("ds_read_b128 v[0:3], v4", "s_waitcnt lgkmcnt(0)", "s_barrier", "s_endpgm")) == []
    assert reads_at_barriers(code("ds_read_b128 v[0:3], v4", "ds_write_b32 v0, v1", "s_waitcnt lgkmcnt(1)", "s_barrier",
                                  "s_endpgm")) == []
    # around a loop: the barrier at its top, the read at its bottom
    back = code("s_waitcnt lgkmcnt(0)", "s_barrier", "ds_read_b128 v[0:3], v4", "s_cbranch_scc1 x", "s_endpgm")
    back[3] = (12, "s_cbranch_scc1", "", 4)
    assert reads_at_barriers(back) == [4]


@pytest.mark.parametrize("kernel", ["linear_int8_rows_kernel", "linear_int8_kernel", "linear_int8_direct_kernel",
                                    "masked_attention_kernel", "masked_attention_join_kernel"])
def test_no_lds_read_in_flight_at_a_barrier(kernels, kernel):
    mine = {n: c for n, c in kernels.items() if re.search(rf"\d{kernel}I", n) and not n.endswith(".kd")}
    assert mine
    bad = {n: [hex(a) for a in reads_at_barriers(c)] for n, c in mine.items()}
    assert not {n: a for n, a in bad.items() if a}

"""Wait states around the loads to LDS that are written in inline asm, in the
built library's own machine code.

The compiler inserts the wait states that gfx9 asks software for, but none
into an asm string.  The loads to LDS take their LDS address from M0 and their
buffer resource and offset from scalar registers:

  * scalar write of M0, then a load to LDS: 1 wait state;
  * vector write of a scalar register (v_readfirstlane_b32), then a load that
    reads it: 5 wait states.

Every instruction between the two counts as one wait state, s_nop N as N + 1;
all ways that lead to a load are followed backwards, across branches.
"""

import collections
import os
import re
import subprocess

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(REPO, "torch-spyre_amd", "torch_spyre", "lib", "libspyre_hip.so")
OBJDUMP = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin", "llvm-objdump")

Ins = collections.namedtuple("Ins", "at op args text")


def parse(lines):
    """The functions of a disassembly that load to LDS: (name, [Ins])."""
    name, body, loads = None, [], False
    for line in lines:
        head = re.match(r"[0-9a-f]+ <(.+)>:$", line)
        if head:
            if loads:
                yield name, [instruction(x) for x in body]
            name, body, loads = head[1], [], False
        elif line.startswith("\t") and "//" in line:
            body.append(line)
            loads = loads or " lds" in line
    if loads:
        yield name, [instruction(x) for x in body]


def instruction(line):
    text, _, at = line.partition("//")
    op, _, args = text.strip().partition(" ")
    # (operands by commas; modifiers stand behind the last one's space)
    return Ins(int(at.split(":")[0], 16), op, [a.split()[0] for a in args.split(",") if a.split()],
               line)


def registers(arg):
    """Scalar registers that an operand names."""
    one, many = re.fullmatch(r"s(\d+)", arg), re.fullmatch(r"s\[(\d+):(\d+)\]", arg)
    return {int(one[1])} if one else set(range(int(many[1]), int(many[2]) + 1)) if many else set()


def predecessors(body):
    index = {x.at: i for i, x in enumerate(body)}
    pred = collections.defaultdict(list)
    for i, x in enumerate(body):
        if x.op.startswith(("s_cbranch", "s_branch")):
            to = re.search(r"<[^>]*?(?:\+0x([0-9a-f]+))?>\s*$", x.text)
            pred[index[body[0].at + int(to[1] or "0", 16)]].append(i)
        if i + 1 < len(body) and x.op not in ("s_branch", "s_endpgm"):
            pred[i + 1].append(i)
    return pred


def before(body, pred, load, states):
    """Instructions with fewer than `states` wait states to body[load]."""
    seen, todo = {}, [(i, 0) for i in pred[load]]
    while todo:
        i, waited = todo.pop()
        if waited >= states or seen.get(i, states) <= waited:
            continue
        seen[i] = waited
        step = int(body[i].args[0], 0) + 1 if body[i].op == "s_nop" else 1
        todo += [(j, waited + step) for j in pred[i]]
    return [body[i] for i in seen]


def is_load(x):
    return x.op.startswith(("buffer_load", "global_load", "scratch_load")) and " lds" in x.text


def early_m0(body):
    """Loads to LDS right behind a scalar write of M0."""
    pred = predecessors(body)
    return [(y.text, x.text) for i, x in enumerate(body) if is_load(x)
            for y in before(body, pred, i, 1) if y.op.startswith("s_") and y.args[:1] == ["m0"]]


def early_scalars(body):
    """Loads to LDS that read a scalar register which a vector instruction has
    just written."""
    pred = predecessors(body)
    return [(y.text, x.text) for i, x in enumerate(body) if is_load(x)
            for y in before(body, pred, i, 5) if y.op.startswith("v_")
            # (carry and condition results stand second)
            and set().union(*map(registers, y.args[:2] if "_co_" in y.op else y.args[:1]))
            & set().union(*map(registers, x.args))]


def listing(*ops):
    return ["0000 <kernel>:"] + [f"\t{op}   // {4 * i:012X}: 00000000" for i, op in enumerate(ops)]


def bodies(lines):
    return [body for _, body in parse(lines)]


def test_scan_finds_missing_wait_states():
    load = "buffer_load_dwordx4 v1, s[4:7], s9 offen lds"
    assert len(early_m0(*bodies(listing("s_mov_b32 m0, s8", load, "s_endpgm")))) == 1
    assert not early_m0(*bodies(listing("s_mov_b32 m0, s8", "s_nop 0", load, "s_endpgm")))
    # over a branch back to the load
    loop = listing("s_branch 1", "s_nop 0", load, "s_mov_b32 m0, s8", "s_cbranch_scc1 65532")
    loop[1] = loop[1] + " <kernel+0x8>"
    loop[5] = loop[5] + " <kernel+0x8>"
    assert not early_m0(*bodies(loop))  # the branch is a wait state
    late = ("v_readfirstlane_b32 s6, v1", "s_mov_b32 m0, s8")
    for nop, found in ((0, 1), (2, 1), (3, 0)):
        assert len(early_scalars(*bodies(listing(*late, f"s_nop {nop}", load)))) == found
    assert not early_scalars(*bodies(listing("v_readfirstlane_b32 s8, v1", "s_nop 0", load)))
    assert not bodies(listing("buffer_load_dwordx4 v[0:3], v4, s[4:7], 0 offen", "s_endpgm"))


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    if not os.path.exists(OBJDUMP):
        pytest.skip("no llvm-objdump")
    d = tmp_path_factory.mktemp("code")
    os.symlink(LIB, d / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=d, check=True, capture_output=True)
    found = []
    for f in sorted(d.iterdir()):
        if "gfx950" in f.name:
            p = subprocess.Popen([OBJDUMP, "-d", "--mcpu=gfx950", "--no-show-raw-insn", str(f)],
                                 stdout=subprocess.PIPE, text=True)
            found += parse(p.stdout)
            assert p.wait() == 0
    assert any("gemm_fp8_ring" in n for n, _ in found) and any("attn" in n for n, _ in found)
    return found


def test_m0_is_written_a_wait_state_ahead(kernels):
    bad = [(name, *pair) for name, body in kernels for pair in early_m0(body)]
    assert not bad, f"{len(bad)} loads, first: {bad[0]}"


def test_scalars_are_written_five_wait_states_ahead(kernels):
    bad = [(name, *pair) for name, body in kernels for pair in early_scalars(body)]
    assert not bad, f"{len(bad)} loads, first: {bad[0]}"

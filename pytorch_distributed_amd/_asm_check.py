"""Checks the compiler's gfx950 assembly of kernels with inline assembly that the compiler cannot wait for.

LDS reads. Such a read names its destination registers as an asm output, which the compiler takes as written at once; the
value arrives later, when an ``s_waitcnt lgkmcnt(n)`` in another asm block has let it. Nothing in the source keeps
the compiler from using a register in between: from copying it, spilling it, or, where the value is unused, from
keeping something else there. What it made of the source can be read, though: ``unawaited_reads`` follows every
path through every kernel and names each instruction that touches the destination of an LDS read before a wait
has covered it. The build refuses kernels for which it finds one.

LDS operations of a wave finish in order, so a read has arrived at ``lgkmcnt(n)`` once n younger ones have been
issued. (Scalar loads share the counter and finish in any order. They only make a wait stricter: with the read
outstanding, so are all younger LDS operations, and the counter is above their number.)

Matrix products. For a product written as inline assembly the compiler inserts no wait states in front of what touches
its result, and it may put a copy of the accumulators anywhere. ``early_products`` names each instruction that touches
the result of such a product, other than a product accumulating into it, before ``WAIT_STATES`` instructions (an
``s_nop n`` counts n + 1) have gone by, on any path.
"""
from __future__ import annotations

import re
from typing import Dict, List, Tuple

_LABEL = re.compile(r"^([A-Za-z_.$][\w.$]*):")
_REGISTER = re.compile(r"(?<![\w\[.])([va])(?:(\d+)|\[(\d+):(\d+)\])(?!\w)")
_RETURNING = re.compile(r"^ds_(read|load|bpermute|permute|swizzle|condxchg|consume|append|ordered_count|\w+_rtn)")
WAIT_STATES = 20  # of the longest (16-pass) product's result for another instruction: 19, and one to spare
_MOST = 15  # the counter's largest value: an age beyond it cannot be told from it

Instruction = Tuple[int, str, str]  # line, mnemonic, operands
State = Dict[Tuple[str, int], int]  # register whose value is on its way -> LDS operations issued since its read


def _registers(text: str):
    found = set()
    for kind, one, first, last in _REGISTER.findall(text):
        found.update((kind, r) for r in (range(int(one), int(one) + 1) if one else range(int(first), int(last) + 1)))
    return found


def _kernels(assembly: str):
    """Name and code of each function: instructions, and labels as (line, ":", label)."""
    name, code, inside = "", [], False
    for number, line in enumerate(assembly.splitlines(), 1):
        line = line.split(";", 1)[0].split("//", 1)[0].rstrip()
        label = _LABEL.match(line)
        if label and not label.group(1).startswith(".L"):
            if code:
                yield name, code
            name, code, inside = label.group(1), [], True
        elif label and label.group(1).startswith(".Lfunc_end"):
            if code:
                yield name, code
            code, inside = [], False
        elif label and inside:
            code.append((number, ":", label.group(1)))
        elif inside and line[:1] in "\t " and line.strip() and not line.strip().startswith("."):
            words = line.split(None, 1)
            code.append((number, words[0], words[1] if len(words) > 1 else ""))
    if code:
        yield name, code


def _blocks(code: List[Instruction]):
    """Basic blocks [(instructions, successors)], the first one the entry."""
    starts, after_jump = [], True
    for i, (_, op, _) in enumerate(code):
        if op == ":" or after_jump:
            starts.append(i)
        after_jump = op.startswith(("s_cbranch", "s_branch", "s_endpgm", "s_setpc"))
    at_label = {code[i][2]: n for n, i in enumerate(starts) if code[i][1] == ":"}
    blocks = []
    for n, i in enumerate(starts):
        body = code[i:starts[n + 1] if n + 1 < len(starts) else len(code)]
        _, op, arg = body[-1]
        follows = [] if op in ("s_branch", "s_endpgm") or n + 1 == len(starts) else [n + 1]
        if op.startswith(("s_cbranch", "s_branch")):
            follows.append(at_label[arg.strip()])
        blocks.append((body, follows))
    return blocks


def _wait(operands: str):
    """The lgkmcnt an s_waitcnt asks for, or None."""
    m = re.search(r"lgkmcnt\((\d+)\)", operands)
    if m:
        return int(m.group(1))
    if re.fullmatch(r"0x[0-9a-fA-F]+|\d+", operands.strip()):
        return (int(operands, 0) >> 8) & 15
    return None


def _run(body: List[Instruction], state: State, report) -> State:
    state = dict(state)
    for line, op, operands in body:
        if op == ":":
            continue
        if op == "s_waitcnt":
            n = _wait(operands)
            if n is not None:
                state = {r: age for r, age in state.items() if age < n}
            continue
        if op.startswith(("s_setpc", "s_swappc", "s_call")):
            report(line, op, "leaves the kernel's code")
        touched = _registers(operands) if state or op.startswith("ds_") else set()
        early = touched & state.keys()
        if early:
            report(line, op, "touches " + ", ".join(f"{k}{n}" for k, n in sorted(early)) + " before the LDS read of it is awaited")
            for r in early:  # once is enough
                del state[r]
        if op.startswith("ds_"):
            for r in state:
                state[r] = min(state[r] + 1, _MOST)
            if _RETURNING.match(op):
                state.update((r, 0) for r in _registers(operands.split(",", 1)[0]))
    return state


def _check(name: str, code: List[Instruction], run, most: int) -> Dict[int, str]:
    """Runs `run(body, state, report) -> state` along every path of a kernel until the states at the blocks' starts (the
    union over the paths, with the least age of each register) stand still. What it reports there, by line."""
    blocks = _blocks(code)
    entry: List[State] = [None] * len(blocks)
    entry[0], work = {}, [0]
    while work:
        n = work.pop()
        body, follows = blocks[n]
        out = run(body, entry[n], lambda *a: None)
        for f in follows:
            old = entry[f]
            new = dict(out) if old is None else {r: min(old.get(r, most), out.get(r, most)) for r in old.keys() | out.keys()}
            if new != old:
                entry[f] = new
                work.append(f)
    found: Dict[int, str] = {}
    for n, (body, _) in enumerate(blocks):
        if entry[n] is not None:
            run(body, entry[n], lambda line, op, what: found.setdefault(line, f"{name}:{line}: {op} {what}"))
    return found


def _listed(found: Dict[int, str]) -> List[str]:
    return [found[line] for line in sorted(found)]


def unawaited_reads(assembly: str) -> List[str]:
    """LDS reads whose registers are touched too early, one line each: ``kernel:line: instruction ...``."""
    return [f for name, code in _kernels(assembly) for f in _listed(_check(name, code, _run, _MOST))]


def early_products(assembly: str) -> List[str]:
    """Inline matrix products whose results are touched too early, likewise."""
    inline, inside = set(), False
    for number, line in enumerate(assembly.splitlines(), 1):
        if "ASMSTART" in line:
            inside = True
        elif "ASMEND" in line:
            inside = False
        elif inside and line.strip().startswith("v_mfma"):
            inline.add(number)

    def run(body, state, report):
        state = dict(state)  # register of a product's result -> wait states since
        for line, op, operands in body:
            if op == ":":
                continue
            if op == "s_nop":
                passed = int(operands, 0) + 1
            else:
                passed = 1
                touched = _registers(operands) if state else set()
                if op.startswith("v_mfma"):  # as its accumulator a product takes another's result in its own time
                    result, a, b = (_registers(o) for o in operands.split(",")[:3])
                    touched = (touched - result) | a | b
                early = touched & state.keys()
                if early:
                    report(line, op, "touches " + ", ".join(f"{k}{n}" for k, n in sorted(early)) + " before the product into it is done")
            state = {r: age + passed for r, age in state.items() if age + passed < WAIT_STATES}
            if line in inline:
                state.update((r, 0) for r in _registers(operands.split(",", 1)[0]))
        return state

    return [f for name, code in _kernels(assembly) for f in _listed(_check(name, code, run, WAIT_STATES))]


def kernels_with_lds_reads(assembly: str) -> List[str]:
    return [name for name, code in _kernels(assembly) if any(op.startswith("ds_read") for _, op, _ in code)]

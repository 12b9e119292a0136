#!/usr/bin/env python3
"""Checks the assembly of a unit whose matrix instructions stand in inline asm.

The products' 256-tiles keep their sums in accumulation registers that nothing but their inline
matrix instructions may touch, and the compiler puts no wait states before inline asm.  So, for each
kernel that has such instructions, in the text that was built:

  * between the first and the last of them no other instruction names an accumulation register;
  * no vector instruction writes a register within 4 wait states before one that reads it, also
    across a loop's end (the hardware wants 2; loads are waited for by count, which the compiler
    does for inline asm too);
  * the sums' first values are written 4 wait states before the first, and the sums are read 19
    after the last (the longest matrix instructions want that many, these fewer).

    check_pinned.py FILE.s KERNELS     exit status 1 unless FILE.s has KERNELS of them, all clean
"""
import re
import sys

BEFORE, BEHIND = 4, 19


def registers(operand):
    """{(file, number)} that an operand names"""
    m = re.match(r"\s*([va])\[(\d+):(\d+)\]", operand)
    if m:
        return {(m.group(1), n) for n in range(int(m.group(2)), int(m.group(3)) + 1)}
    m = re.match(r"\s*([va])(\d+)\b", operand)
    return {(m.group(1), int(m.group(2)))} if m else set()


def kernels(text):
    """{name: [(mnemonic, operands, inline)]}, labels as ("label", [name], False)"""
    out, body, inline = {}, None, False
    for line in text.split("\n"):
        if "#ASMSTART" in line:
            inline = True
        elif "#ASMEND" in line:
            inline = False
        code = line.split(";")[0].strip()
        m = re.match(r"([\w.$]+):", code)
        if m:
            if not m.group(1).startswith((".", "$")):
                body = out.setdefault(m.group(1), [])
            elif body is not None:
                body.append(("label", [m.group(1)], False))
        elif code and not code.startswith(".") and body is not None:
            name, _, rest = code.partition(" ")
            body.append((name, rest.split(",") if rest else [], inline))
    return out


def states(name, operands):
    if name == "label":
        return 0
    return int(operands[0].split()[0], 0) + 1 if name == "s_nop" else 1


def writes(name, operands):
    """registers that a vector instruction writes"""
    return registers(operands[0]) if name.startswith("v_") and operands else set()


def check(body):
    """What is wrong with a kernel's instructions, None where it has no pinned ones."""
    pinned = [n for n, (name, ops, inline) in enumerate(body)
              if inline and name.startswith("v_mfma") and ops[0].strip().startswith("a")]
    if not pinned:
        return None
    wrong, own = [], set(pinned)
    sums = set().union(*(registers(body[n][1][0]) for n in pinned))
    for n in range(pinned[0], pinned[-1] + 1):
        name, ops, _ = body[n]
        if n not in own and name != "label" and any(r[0] == "a" for o in ops for r in registers(o)):
            wrong.append(f"{name} {','.join(ops)} touches the sums")
    jumps = {}
    for n, (name, ops, _) in enumerate(body):
        if name.startswith("s_cbranch") or name == "s_branch":
            jumps.setdefault(ops[0].strip(), []).append(n)

    def back(n, left, need, seen):
        """walk back from before instruction n for `left` wait states"""
        while n >= 0 and left > 0:
            name, ops, _ = body[n]
            if name in ("s_branch", "s_endpgm"):  # not reached by falling through
                return
            if name == "label":
                for j in jumps.get(ops[0], ()):
                    if (j, left) not in seen:
                        seen.add((j, left))
                        step(j, left, need, seen)
            elif n not in own and writes(name, ops) & need:
                wrong.append(f"{name} {','.join(ops)} right before a matrix instruction reads it")
                return
            left -= states(name, ops)
            n -= 1

    def step(j, left, need, seen):  # the branch itself is one wait state
        back(j - 1, left - 1, need, seen)

    for n in pinned:
        need = set().union(*(registers(o) for o in body[n][1][1:3]))
        back(n - 1, BEFORE, need, set())
    back(pinned[0] - 1, BEFORE, sums, set())
    gap = 0
    for name, ops, _ in body[pinned[-1] + 1:]:
        if name != "label" and any(registers(o) & sums for o in ops):
            break
        gap += states(name, ops)
    if gap < BEHIND:
        wrong.append(f"the sums are read {gap} wait states behind the last matrix instruction")
    return wrong


def main(path, count):
    with open(path) as f:
        found = {name: check(body) for name, body in kernels(f.read()).items()}
    found = {name: wrong for name, wrong in found.items() if wrong is not None}
    for name, wrong in found.items():
        for line in wrong[:5]:
            print(f"{name}: {line}")
    if len(found) != count:
        print(f"{path}: {len(found)} kernels with pinned sums, not {count}")
    return int(len(found) != count or any(found.values()))


if __name__ == "__main__":
    sys.exit(main(sys.argv[1], int(sys.argv[2])))

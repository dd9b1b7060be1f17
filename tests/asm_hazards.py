"""Reads of a matrix instruction's result that come too soon, in the assembly of a kernel file.

The hardware does not hold back an instruction that reads a register which a matrix instruction
is still writing: the compiler has to put enough wait states between them.  It has left them out
once where a branch led straight from the instruction to the read (hipcc of ROCm 7.2, results
in accumulation registers).  This walks every path from each matrix instruction."""
import re

# Wait states before a vector or memory instruction may read the result: passes + 3 for 16-bit
# operands (4 passes for 16x16x32, 8 for 32x32x16), passes + 2 for 16x16x4 fp32 (8 passes).
NEED = {"v_mfma_f32_16x16x32_bf16": 7, "v_mfma_f32_16x16x32_f16": 7,
        "v_mfma_f32_16x16x4_f32": 10}


def _registers(operand):
    m = re.match(r"-?\|?([av])\[(\d+):(\d+)\]", operand)
    if m:
        return {m.group(1) + str(i) for i in range(int(m.group(2)), int(m.group(3)) + 1)}
    m = re.match(r"-?\|?([av])(\d+)", operand)
    return {m.group(1) + m.group(2)} if m else set()


def _operands(text):
    parts = text.split(None, 1)
    return parts[0], [o.strip() for o in re.split(r",(?![^\[]*\])", parts[1])] if parts[1:] else []


def _functions(text):
    name, found = None, {}
    for line in text.splitlines():
        m = re.match(r"(_Z\w+):", line)
        if m:
            name = m.group(1)
            found[name] = []
        elif re.match(r"\s*\.section|\.Lfunc_end", line):
            name = None
        elif name:
            m = re.match(r"(\.LBB\w+):", line)
            code = line.split(";")[0].strip()
            if m:
                found[name].append(m.group(1) + ":")
            elif code and not code.startswith("."):
                found[name].append(code)
    return found


def early_reads(text):
    """(number of matrix instructions, what reads one's result too soon)."""
    count, early = 0, []
    for name, code in _functions(text).items():
        at = {c[:-1]: i for i, c in enumerate(code) if c.endswith(":")}
        for start, first in enumerate(code):
            if not first.startswith("v_mfma"):
                continue
            count += 1
            op, ops = _operands(first)
            written, need = _registers(ops[0]), NEED[op]
            paths, seen = [(start + 1, 0)], set()
            while paths:
                i, waited = paths.pop()
                while i < len(code) and waited < need and (i, waited) not in seen:
                    seen.add((i, waited))
                    if code[i].endswith(":"):
                        i += 1
                        continue
                    op, ops = _operands(code[i])
                    if op == "s_endpgm":
                        break
                    if op == "s_branch":
                        i, waited = at[ops[0]], waited + 1
                        continue
                    if op.startswith("s_cbranch"):
                        paths.append((at[ops[0]], waited + 1))
                    elif op.startswith("v_mfma"):
                        if written & _registers(ops[0]):
                            break  # goes on in the same registers: the hardware holds it back
                    elif op.startswith(("v_", "ds_", "global_", "buffer_", "flat_", "scratch_")):
                        stores = ("ds_write", "global_store", "buffer_store", "flat_store",
                                  "scratch_store", "v_cmp", "v_permlane")
                        read = set().union(*map(_registers, ops if op.startswith(stores)
                                                else ops[1:]), set())
                        if read & written:
                            early.append(f"{name}: {first} -> {code[i]} after {waited}")
                            break
                    waited += int(ops[0], 0) + 1 if op == "s_nop" else 1
                    i += 1
    return count, early

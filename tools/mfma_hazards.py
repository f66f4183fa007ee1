#!/usr/bin/env python3
"""Look for matrix-instruction results that are read too early in `hipcc -S` listings.

A gfx950 v_mfma writes its registers several wait states after it issues, and the hardware does not interlock a vector,
LDS or memory instruction that reads them before: the compiler inserts the waits.  It has been seen to leave them out where
the first reader is the first instruction of a block that a branch right behind the v_mfma leads to, which gives wrong
values.  This follows every path from every v_mfma over branches, results in ordinary and in accumulation registers, and
reports readers closer than the states the product needs: its passes (a quarter of its cycles) + 3, on gfx950 one more (8 for a
16x16x32 product of 16-bit values, the shortest distance in the compiler's own code).  The target is the one that the listing names.

    hipcc --offload-arch=gfx950 <the build's flags> --cuda-device-only -S file.hip -o file.s && tools/mfma_hazards.py file.s
"""
import re
import sys

PASSES = {"16x16x16": 4, "16x16x32": 4, "32x32x8": 8, "32x32x16": 8}
REG = re.compile(r"\b([va])(?:(\d+)\b|\[(\d+):(\d+)\])")


def registers(operands: str) -> set:
    out = set()
    for m in REG.finditer(operands):
        first, last = (m.group(2), m.group(2)) if m.group(2) else (m.group(3), m.group(4))
        out.update((m.group(1), i) for i in range(int(first), int(last) + 1))
    return out


def need(mfma: str, target: str) -> int:
    """States between a product and the first instruction that may read its result (shapes unknown: 16 passes)."""
    passes = next((n for shape, n in PASSES.items() if re.search(rf"_{shape}(?!\d)", mfma.split()[0])), 16)
    return passes + 3 + (target == "gfx950")


def kernels(path: str) -> dict:
    """{kernel: [("target", name), then ("label", name) | ("ins", text)]}"""
    found, cur, target = {}, None, ""
    for line in open(path):
        m = re.match(r"^(_Z\w+):", line)
        if m:
            cur = found.setdefault(m.group(1), [("target", target)])
        elif ".amdgcn_target" in line:
            target = re.search(r"gfx\w+", line).group(0)
        elif cur is not None:
            m = re.match(r"^(\.L\w+):", line)
            text = line.split(";")[0].strip()
            if ".end_amdhsa_kernel" in line:
                cur = None
            elif m:
                cur.append(("label", m.group(1)))
            elif text and not text.startswith("."):
                cur.append(("ins", text))
    return found


def early_reads(code: list) -> list:
    """(v_mfma, reader, wait states between them) of one kernel, for all readers that come too early."""
    target = code[0][1]
    labels = {name: i for i, (kind, name) in enumerate(code) if kind == "label"}
    bad = []
    for start, (kind, text) in enumerate(code):
        if kind != "ins" or not text.startswith("v_mfma"):
            continue
        written, states = registers(text.split(",")[0].split(None, 1)[1]), need(text, target)
        paths, seen = [(start + 1, 0)], {}
        while paths:
            i, waited = paths.pop()
            while i < len(code) and waited < states and seen.get(i, states) > waited:
                seen[i] = waited
                kind, ins = code[i]
                i += 1
                if kind == "label":
                    continue
                op = ins.split()[0]
                if op == "s_endpgm":
                    break
                if op == "s_nop":
                    waited += int(ins.split()[1]) + 1
                    continue
                if op.startswith(("s_cbranch", "s_branch")):
                    if ins.split()[-1] in labels:
                        paths.append((labels[ins.split()[-1]], waited + 1))
                    if op == "s_branch":
                        break
                elif op.startswith("v_mfma"):
                    if registers(ins[len(op):]) & written:
                        break  # (chains of matrix instructions have rules of their own)
                elif op.startswith(("v_", "ds_", "buffer_", "global_", "flat_", "scratch_")) and registers(ins[len(op):]) & written:
                    bad.append((text, ins, waited))
                    break
                waited += 1
    return bad


def main(paths) -> int:
    count = 0
    for path in paths:
        for name, code in kernels(path).items():
            for mfma, reader, waited in early_reads(code):
                count += 1
                print(f"{name}: {mfma}  ->  {reader}  after {waited} of {need(mfma, code[0][1])} wait states")
    print(f"{count} results read too early")
    return 1 if count else 0


if __name__ == "__main__":
    sys.exit(main(sys.argv[1:]))

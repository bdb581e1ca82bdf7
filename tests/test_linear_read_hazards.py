"""The hand-placed LDS reads of the linear layers' kernels (ds_read_b128; ds_read_b64_tr_b16 in the weight gradient) follow the
protocol that test_lds_read_hazards.py states: no instruction touches a destination between a read and the wait that covers it,
nothing is in flight at a loop edge.  Their loops keep everything in registers: no memory of a lane's own is touched between two
multiplies of a loop."""
import os
import re
import subprocess

import pytest

import test_lds_read_hazards as H


def _functions(source):
    subprocess.run(["make", "-C", H.CSRC, "-j3", "isa-linear"], check=True, stdout=subprocess.DEVNULL, stderr=subprocess.DEVNULL)
    current = None
    with open(os.path.join(H.CSRC, "build", source + ".s")) as f:
        for no, raw in enumerate(f, 1):
            m = re.match(r"^(_Z\w+):\s*(;.*)?$", raw)
            if m:
                name, current = m.group(1), []
            elif raw.startswith(".Lfunc_end") and current is not None:
                yield name, current
                current = None
            elif current is not None:
                current.append((no, raw))


@pytest.mark.parametrize("source,least", [("linear_bf16", 20), ("linear_f32", 16), ("linear_wgrad", 6)])
def test_operand_reads(source, least):
    kernels, total, problems = 0, 0, []
    for name, lines in _functions(source):
        if not any(op in raw for _, raw in lines for op in ("ds_read_b128", "ds_read_b64_tr_b16")):
            continue
        lines = [(no, raw.replace("ds_read_b64_tr_b16", "ds_read_b128")) for no, raw in lines]
        seen, bad = H.check_function(name, lines)
        kernels, total = kernels + 1, total + seen
        problems += bad
        # blocks that multiply: four at least, and no scratch
        block, multiplies = [], 0
        for no, raw in lines + [(0, ".Lend:")]:
            if raw.strip().startswith(".L") and raw.strip().endswith(":"):
                if multiplies >= 4 and any("scratch_" in r for _, r in block):
                    problems.append(f"{name}: scratch between multiplies, line {block[0][0]}")
                block, multiplies = [], 0
            elif raw.strip():
                block.append((no, raw))
                multiplies += "v_mfma" in raw
    assert kernels >= least and total >= 100, (kernels, total)
    assert not problems, "\n".join(problems[:20])

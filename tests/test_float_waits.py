"""The waits of the float experts' products: a role of the kernel may only wait
with a limit, since another role that gave up may never come.  Checked on the
source: a wait that runs out cannot be provoked from outside, and a kernel that
hangs may not be run."""

import re
from pathlib import Path

SOURCE = Path(__file__).resolve().parent.parent / "distributedmoellm_b200" / "csrc" / "mb_grouped.cu"

# barriers of a CTA, of some of its warps or of a cluster: none has a limit
UNBOUNDED = re.compile(r"__syncthreads|cluster_sync|mb_named_barrier|bar\.sync|barrier\.")


def code(text):
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", text, flags=re.S)


def section(text, start, end):
    a = text.index(start)
    return text[a:text.index(end, a)]


def test_roles_wait_with_a_limit_only():
    text = code(SOURCE.read_text())
    epilogue = section(text, "struct Epilogue {", "__global__")
    roles = section(text, "const int split = wsum[31];", "if (warp == Role::kMma) tc_dealloc")
    roles = roles[:roles.rindex("tc_before();")]           # what follows is the CTA's barrier at the end
    assert "ep.item(" in roles and "tc_mma_ss" in roles and "tma_load2" in roles
    for name, part in (("epilogue", epilogue), ("roles", roles)):
        assert not UNBOUNDED.findall(part), name


def test_lanes_of_a_warp_give_up_together():
    """A whole warp's wait for an item ends in one vote: lanes that leave a loop alone would miss the others' warp-wide steps."""
    pop = section(code(SOURCE.read_text()), "bool pop(Item& v)", "return v.nrows > 0;")
    assert re.search(r"if \(WARP\) got = __all_sync\(0xffffffffu, got\);\s+if \(!got\) return false;", pop)


def test_work_in_flight_ends_before_the_cta():
    """The loads and the products wait, with a limit, for what they issued last, whatever made them stop: a copy, or a
    product's arrival, behind the CTA's end would reach the shared memory of the next one."""
    text = code(SOURCE.read_text())
    loads = section(text, "if (warp == Role::kLoad) {", "} else if (warp == Role::kMma) {")
    mma = section(text, "} else if (warp == Role::kMma) {", "} else if (warp == Role::kFind) {")
    for part, bar in ((loads, r"fullb \+ 8 \* st\.slot, st\.full_parity\(\)"), (mma, r"mb_smem_addr\(mma_done\), 0")):
        loop = section(part, "while (ok && ring.pop<false>(w))", "__syncwarp();")
        end = re.search(r"n < kDrainTries && !bar_try\(" + bar, loop)
        assert end and "abort_flag)" not in loop[loop.rindex("++issued;" if part is loads else "part = 0;"):end.start()]

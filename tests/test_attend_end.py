"""What the attention's CTAs do before they end when a wait has expired, read from the source: what is in flight is waited for behind
the barrier where all roles meet. A role that looks on its own way out does not see the wait of another role expire after it."""
import os
import re

import amd_developer_challenge_2025_b200 as pkg


def attend_kernel():
    with open(os.path.join(os.path.dirname(pkg.__file__), "csrc", "mla_cache_sm100.cu")) as f:
        code = re.sub(r"//[^\n]*", "", f.read())
    begin = code.index("attend_kernel(const __grid_constant__ CUtensorMap")
    return code[begin:code.index("\n}\n", begin)]


def test_copies_and_products_come_to_rest_behind_the_last_barrier():
    roles, end = attend_kernel().rsplit("__syncthreads();", 1)
    assert re.search(r"if \(sh\.expired != 0\)", end)
    for bar in ("sh.full[n]", "sh.q_full", "sh.drained"):
        assert f"at_rest(&{bar}" in end, bar
    assert "umma_commit(smem_u32(&sh.drained))" in end and end.index("drained") < end.index("tcgen05.dealloc")
    assert "sh.drained" not in roles.split("mbar_init(smem_u32(&sh.drained), 1);")[1]
    # copies of the rows' own kind end in the role that issued them, which is their only owner
    assert "cp.async.wait_all" in roles


def test_the_next_kernel_begins_once_tmem_is_allocated():
    """Its CTAs may come to the same SM. One that allocates TMEM before this CTA has its own, and then waits for this kernel's end, would
    never get there."""
    code = attend_kernel()
    alloc, go = code.index("tcgen05.alloc"), code.index("pdl_launch_dependents();")
    assert code.count("pdl_launch_dependents();") == 1 and alloc < go and "__syncthreads();" in code[alloc:go]

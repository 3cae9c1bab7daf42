"""Two warps of a kernel issue products into the tensor pipe, and the one that overwrites the other's operand in TMEM follows it by a counter in
shared memory.  The order holds if the counter is published behind a tcgen05 fence with release, and read with acquire in front of another: a
missing fence need not show in a run, so the sources are what is checked."""
import os
import re

import pytest

from tests.test_dependent_launch_sources import CSRC, functions, strip_comments


@pytest.mark.parametrize("path,kernel", [("cross_attn.cu", "cross_attn_pair_kernel"), ("attn_flash.cu", "attn_flash_pair_kernel")])
def test_the_counter_orders_the_products(path, kernel):
    bodies = {n: b for n, _, b in functions(strip_comments(open(os.path.join(CSRC, path)).read()), r"__global__")}
    body = bodies[kernel]
    # written once at the start, before the block's first barrier, and then by release only
    assert len(re.findall(r"(?<!uint32_t )\*pv_issued\s*=[^=]", body)) == 1 and body.index("*pv_issued = 0") < body.index("__syncthreads")
    publish = [m.start() for m in re.finditer(r"st_release_cta\(pv_issued", body)]
    assert len(publish) == 1
    before = body[:publish[0]]
    assert before.rindex("tc_fence_before()") > before.rindex("mma_f16_tmem_a_pair(")
    # read by acquire only, and the products that rely on it stand behind a fence
    assert not re.findall(r"\*pv_issued\s*[<>]", body)
    reads = [m.start() for m in re.finditer(r"ld_acquire_cta\(pv_issued", body)]
    assert len(reads) >= 2
    after = body[reads[-1]:]
    assert after.index("tc_fence_after()") < re.search(r"mma_f16_pair\(|issue_s\(", after).start()

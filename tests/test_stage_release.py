"""A stage that TMA fills and warps read with ordinary loads goes back to the loader behind a proxy fence: an mbarrier's arrive orders such reads
against other ordinary accesses only, not against the next fill.  Reads of the next fill need not show in a run, so the source is checked."""
import os
import re

import pytest

from tests.test_dependent_launch_sources import CSRC, functions, strip_comments


def test_stages_read_by_ldmatrix_are_released_behind_the_fence():
    bodies = {n: b for n, _, b in functions(strip_comments(open(os.path.join(CSRC, "cross_attn.cu")).read()), r"__global__")}
    body = bodies["cross_few_kernel"]
    releases = [m.start() for m in re.finditer(r"mbar_arrive\(&(?:free_|q_free)\[", body)]
    assert len(releases) == 2
    for at in releases:
        before = body[:at]
        last_read = before.rindex("xf_ldmatrix")
        fence = before.rindex("fence_proxy_async_smem()")
        # every lane's own fence, then all of them together, then one arrives
        assert last_read < fence < before.rindex("__syncwarp()"), body[at:at + 40]


@pytest.mark.gpu
@pytest.mark.parametrize("B,S,n_q,n_kv,hd,cap", [(700, 1, 8, 1, 256, 512), (500, 2, 8, 2, 128, 640), (900, 1, 3, 1, 64, 768), (2, 1, 8, 1, 256, 64 * 700)])
def test_clean_blocks_of_many_units_repeat_their_bits(B, S, n_q, n_kv, hd, cap):
    """Stages refilled over and over with nothing hidden, so that no other fence stands between the reads and the fill."""
    from tests.gpu_util import require_cuda
    from tests.test_cross_attention import check
    from tests.test_key_mass import make

    torch = require_cuda()
    import vla_cpp_b200 as vb

    lens = [cap - 64 * (b % 5) for b in range(B)]
    st, q, lens, _, _ = make(torch, B, S, n_q, n_kv, hd, cap, lens, False, 41, layers=1)
    out, lse = vb.cross_attention(st, 0, q, lens=lens)
    assert vb.device_status() == 0
    check(torch, st, 0, q, lens, None, out, lse)
    for _ in range(30):
        again = vb.cross_attention(st, 0, q, lens=lens)
        assert torch.equal(again[0], out) and torch.equal(again[1], lse)

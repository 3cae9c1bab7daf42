"""Kernels whose products come from two warps: P lies over its S in TMEM, so the S of a later block may be issued only when the P V that reads those
weights is complete.  The tensor pipe keeps the order of one warp's products, not of two warps'; that one was issued behind the other is not
enough, whatever fences stand in between."""
import os

import pytest

from tests.test_dependent_launch_sources import CSRC, functions, strip_comments


@pytest.mark.parametrize("path,kernel,wait", [("cross_attn.cu", "cross_attn_pair_kernel", "warp_wait(&pv_done["),
                                              ("attn_flash.cu", "attn_flash_pair_kernel", "mbar_wait(&pv_done[")])
def test_scores_wait_for_the_commit_of_the_product_that_reads_the_weights(path, kernel, wait):
    bodies = {n: b for n, _, b in functions(strip_comments(open(os.path.join(CSRC, path)).read()), r"__global__")}
    issuer = bodies[kernel]
    issuer = issuer[issuer.index("constexpr uint32_t idesc_s"):]
    issuer = issuer[:issuer.index("constexpr uint32_t idesc_o")]  # the warp that issues S
    at = issuer.index(wait)  # parity: of the block that used this buffer before
    statement = issuer[at:issuer.index(";", at)]
    assert "& 1u) ^ 1u" in statement and "NS" in statement
    assert "tc_fence_after()" in issuer[at:]
    committed = bodies[kernel]
    committed = committed[committed.index("constexpr uint32_t idesc_o"):]
    assert committed.index("mma_f16_tmem_a_pair(") < committed.index("tc_commit_pair(&pv_done[")


def leftovers(torch):
    """Another kernel's use of the SMs, and an L2 without the call's operands, in front of a call."""
    junk = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    return lambda: junk.random_()


@pytest.mark.gpu
@pytest.mark.parametrize("hd,split", [(256, True), (256, False), (128, True), (64, True)])
def test_cross_attention_behind_other_kernels(hd, split):
    """Pieces of one to four blocks, hidden ranges that cover whole blocks: the same bits as the first time, call after call."""
    from tests.gpu_util import require_cuda
    from tests.test_cross_attention import check
    from tests.test_key_mass import make

    torch = require_cuda()
    import vla_cpp_b200 as vb

    lens = [1789, 2438, 768, 941, 896, 1552, 423, 757, 1792, 606, 241]
    pads = [(1090, 1675), (1548, 1751), (87, 218), (246, 619), (57, 116), (1206, 1213), (394, 415), (139, 257), (921, 1121), (193, 224), (128, 173)]
    st, q, lens, _, _ = make(torch, 11, 4, 24, 3, hd, 2555, lens, False, 9291, layers=1)
    pads = torch.tensor(pads, dtype=torch.int32, device="cuda")
    disturb = leftovers(torch)
    out, lse = vb.cross_attention(st, 0, q, lens=lens, max_len=2438, pad_ranges=pads, split=split)
    check(torch, st, 0, q, lens, pads, out, lse)
    wrong = torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(4000):
        disturb()
        o, l = vb.cross_attention(st, 0, q, lens=lens, max_len=2438, pad_ranges=pads, split=split)
        wrong += (o.view(torch.int16) != out.view(torch.int16)).any() | (l.view(torch.int32) != lse.view(torch.int32)).any()
    assert int(wrong) == 0 and vb.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("hd,B,rows", [(256, 90, 400), (256, 200, 200), (128, 90, 700)])
def test_attention_behind_other_kernels(hd, B, rows):
    from tests.gpu_util import require_cuda

    torch = require_cuda()
    import vla_cpp_b200 as vb

    n_q, S = 8, 51
    g = torch.Generator(device="cuda").manual_seed(hd + B)
    st = vb.KvStore(1, B, 1, hd, rows, 0)
    st.k.normal_(0, 1, generator=g)
    st.v.normal_(0, 1, generator=g)
    q = (torch.randn(B, n_q, S, hd, device="cuda", generator=g) * 1.5).bfloat16()
    disturb = leftovers(torch)
    out = vb.attention(st, 0, q, S, n_q, rows, vb.MASK_NONE)
    wrong = torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(3000):
        disturb()
        wrong += (vb.attention(st, 0, q, S, n_q, rows, vb.MASK_NONE).view(torch.int16) != out.view(torch.int16)).any()
    assert int(wrong) == 0 and vb.device_status() == 0

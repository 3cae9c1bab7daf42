"""The two softmax warps of a row exchange their parts of the row's sum through slots in shared memory.  Between one warp's read of the
other's slot and the next write of that slot the two have to have met, or a warp that was held up reads the sum of a later segment -- a
race that a run need not show, so what is checked is the protocol: every short sequence of segments is walked, with as many sets of slots
as the source has, and the meetings in front of each read and write are counted."""
import itertools
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vla_cpp_b200", "csrc")


def sets_of(path, struct):
    """SUM_SETS of a kernel's shared memory; 1 where there is no such constant."""
    text = open(os.path.join(CSRC, path)).read()
    body = text[text.index(f"struct {struct} {{"):]
    m = re.search(r"\bSUM_SETS = (\d+)", body[:body.index("\n};")])
    if not m:
        return 1
    assert re.search(r"\(u % L::SUM_SETS\)", text)  # a segment's (unit's) number says which
    return int(m.group(1))


def events(segments):
    """(kind, segment) in one warp's order: "meet", "write" and "read" of the row sums of a segment.  A segment is (blocks, whether the warps
    have rows in it): a block is a meeting, for the maxima; behind a segment's first block the one before it is drained.  What drains the last
    one: nothing (a turn without a block)."""
    out = []

    def drain(u):
        if segments[u][1]:
            out.extend([("write", u), ("meet", u), ("read", u)])

    for u, (blocks, live) in enumerate(segments):
        for j in range(blocks):
            if live:
                out.append(("meet", u))
            if j == 0 and u > 0:
                drain(u - 1)
    drain(len(segments) - 1)
    return out


def unordered(seq, sets):
    """Segments whose write is not behind a meeting that follows the last read of its slot."""
    met, last_read, bad = 0, {}, []
    for kind, u in seq:
        if kind == "meet":
            met += 1
        elif kind == "read":
            last_read[u % sets] = met
        elif last_read.get(u % sets, -1) == met:
            bad.append(u)
    return bad


def sequences(with_empty):
    kinds = [(b, live) for b in (1, 2, 3) for live in ((True, False) if with_empty else (True,))]
    for n in range(1, 6):
        yield from itertools.product(kinds, repeat=n)


def test_one_set_is_not_enough():
    """What the protocol did with a single set: the drain of a last segment of one block wrote over sums that nobody is known to have read."""
    assert unordered(events([(3, True), (1, True)]), 1) == [1]
    assert unordered(events([(3, True), (1, True), (2, False)]), 1) == [1]
    assert unordered(events([(3, True), (2, True)]), 1) == []


@pytest.mark.parametrize("path,struct,with_empty", [("cross_attn.cu", "CrossPairSmem", True), ("attn_flash.cu", "FlashPairSmem", False)])
def test_every_write_is_behind_a_meeting(path, struct, with_empty):
    sets = sets_of(path, struct)
    for segments in sequences(with_empty):
        assert not unordered(events(segments), sets), (sets, segments)


@pytest.mark.gpu
@pytest.mark.parametrize("B,S,n_q,n_kv,cap,lens", [
    (170, 40, 8, 1, 128, [128] * 170),                                    # 320 rows: units of one block, the second of an item without rows in the odd CTA
    (120, 51, 8, 1, 300, [(257, 1, 128, 300)[b % 4] for b in range(120)]),  # one block behind three and three behind one
    (300, 17, 4, 1, 100, [(100, 7, 0)[b % 3] for b in range(300)]),       # more observations than are sorted
    (3, 64, 4, 1, 6000, [5900, 129, 128]),                                # pieces of one block
])
def test_segments_of_one_block(B, S, n_q, n_kv, cap, lens):
    from tests.gpu_util import require_cuda
    from tests.test_cross_attention import check
    from tests.test_key_mass import make

    torch = require_cuda()
    import vla_cpp_b200 as vb

    st, q, lens, _, _ = make(torch, B, S, n_q, n_kv, 256, cap, lens, False, 31, layers=1)
    # sums that differ from segment to segment by far more than rounding
    q.mul_(torch.linspace(0.1, 1.0, B, device="cuda").bfloat16()[:, None, None, None])
    for split in (True, False):
        out, lse = vb.cross_attention(st, 0, q, lens=lens, split=split)
        assert vb.device_status() == 0
        check(torch, st, 0, q, lens, None, out, lse)
        for _ in range(20):
            again = vb.cross_attention(st, 0, q, lens=lens, split=split)
            assert torch.equal(again[0], out) and torch.equal(again[1], lse)


@pytest.mark.gpu
@pytest.mark.parametrize("hd,rows", [(256, 128), (256, 100), (128, 97), (256, 129)])
def test_units_of_one_key_block(hd, rows):
    """vlab200_attention over CTA pairs that each walk several units of one block.  Bound: one bf16 rounding of the value, one of each weight
    (2^-8 each), and what is done in 32 bits: a score's sum is off by at most hd 2^-24 sum |q k| scale <= 256 x 2^-24 x 30 < 2^-11, which both a
    weight and the row's sum have: 2^-10; exponentials and sums of 128 terms are far below."""
    from tests.gpu_util import require_cuda

    torch = require_cuda()
    import vla_cpp_b200 as vb

    B, n_q, S = 190, 4, 50  # 200 rows: two tiles, 190 units on 74 pairs
    g = torch.Generator(device="cuda").manual_seed(hd + rows)
    st = vb.KvStore(1, B, 1, hd, rows, 0)
    st.k.normal_(0, 1, generator=g)
    st.v.normal_(0, 1, generator=g)
    q = (torch.randn(B, n_q, S, hd, device="cuda", generator=g) * torch.linspace(0.1, 1.5, B, device="cuda")[:, None, None, None]).bfloat16()
    out = vb.attention(st, 0, q, S, n_q, rows, vb.MASK_NONE)
    p = torch.softmax(q.double() @ st.k[0].double().transpose(-1, -2) * hd ** -0.5, -1)
    fold = lambda t: t.transpose(1, 2).reshape(B, S, n_q * hd)
    want, size = fold(p @ st.v[0].double()), fold(p @ st.v[0].double().abs())
    assert bool(((out.double() - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -10) * size).all())
    for _ in range(20):
        assert torch.equal(vb.attention(st, 0, q, S, n_q, rows, vb.MASK_NONE), out)
    assert vb.device_status() == 0

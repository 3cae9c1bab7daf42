"""cross_attention against its formula in 64 bits.

Bound of an output element: one bf16 rounding of the value (bf16 has 8 significant bits: neighbours lie 2^-7 of a value just above a
power of two apart, half of that is 2^-8 relative); the weights' rounding to bf16 (2^-8 each, the same) and the weights' error in 32 bits (the score's sum hd^1/2 Z 2^-24, the exponent 4 E 2^-24, the exponential 2^-22, together e) on numerator
and sum: (2^-8 + 2 e) sum p |v| -- the sum of weights keeps the unrounded ones -- and the product's sum, (rows + 128) 2^-24 sum p |v|.
lse: e plus the logarithm and its scaling, 4 x 2^-24 (|lse| + 1)."""
import ctypes as C
import math

import pytest

from tests.gpu_util import require_cuda
from tests.test_key_mass import make, scores, visible


def test_argument_checks_need_no_gpu():
    from vla_cpp_b200 import api

    def call(**kw):
        st = api._KvStoreC(*(kw.pop(n, d) for n, d in (("k", 1 << 20), ("v", 2 << 20), ("layers", 1), ("obs", 2), ("n_kv", 1), ("hd", 64),
                                                       ("cap", 8), ("prefix", 0))))
        g = lambda n, d: kw.pop(n, d)
        p = lambda v: C.c_void_p(v) if v else None
        return api.lib().vlab200_cross_attention(C.byref(st), g("layer", 0), p(g("q", 3 << 20)), p(g("out", 4 << 20)), p(g("lse", 5 << 20)), g("S", 1), g("n_q", 2),
                                                 None, g("max_len", 8), None, C.c_float(g("scale", 0.0)), p(g("ws", None)),
                                                 C.c_int64(g("ws_bytes", 0)), None)

    for bad in (dict(k=None), dict(v=None), dict(q=None), dict(out=None), dict(layer=1), dict(layer=-1), dict(S=0), dict(n_q=0), dict(n_q=3, n_kv=2),
                dict(max_len=9), dict(max_len=-1), dict(scale=-1.0), dict(scale=math.nan), dict(q=24), dict(k=8), dict(v=24), dict(out=40),
                dict(ws=16, ws_bytes=1 << 30), dict(ws_bytes=-1), dict(obs=0), dict(cap=0),
                dict(out=3 << 20), dict(out=1 << 20), dict(lse=4 << 20), dict(lse=(2 << 20) + 64)):
        assert call(**bad) == -1, bad
    assert call(hd=80) == -4
    st = api._KvStoreC(16, 16, 1, 2, 2, 64, 8, 0)
    assert api.lib().vlab200_cross_attention_ws_bytes(C.byref(st), 1, 3, 8) == -1
    assert api.lib().vlab200_cross_attention_ws_bytes(C.byref(st), 0, 2, 8) == -1
    assert api.lib().vlab200_cross_attention_ws_bytes(C.byref(st), 1, 2, 9) == -1


CASES = [
    # B, S, n_q, n_kv, hd, cap, lens, pad
    (1, 1, 1, 1, 64, 1, [1], False),
    (1, 1, 20, 5, 128, 1001, [1001], False),            # one token: one block per CTA
    (1, 1, 8, 1, 256, 2000, [1999], False),
    (3, 1, 3, 1, 64, 130, [129, 0, 128], True),
    (4, 50, 15, 5, 64, 241, [241, 0, 113, 127], True),  # 150 rows: a second tile of 22
    (2, 51, 8, 1, 256, 300, [300, 257], True),
    (2, 51, 8, 1, 256, 900, [1, 816], False),
    (2, 33, 4, 1, 128, 400, [400, 385], True),          # 132 rows
    (1, 129, 4, 2, 128, 390, [385], True),              # 258 rows: a second unit of two rows
    (1, 130, 5, 1, 256, 390, [385], False),
    (40, 3, 6, 2, 64, 700, None, True),                 # more than 32 observations
    (70, 9, 4, 2, 128, 300, None, False),
    (40, 40, 8, 2, 256, 500, None, True),
    (5, 300, 2, 2, 64, 1500, None, False),
    (3, 200, 4, 2, 128, 1500, None, True),
    (3, 100, 4, 1, 256, 1500, None, True),
    (300, 2, 2, 2, 64, 200, None, True),                # more observations than are sorted
    (270, 20, 8, 1, 256, 300, None, False),
    (260, 70, 4, 1, 128, 150, None, True),
    (3, 2, 8, 1, 256, 700, None, True),                 # 16 rows: the most that the kernel of few rows takes
    (2, 17, 2, 2, 128, 300, None, True),                # 17
    (5, 1, 4, 4, 128, 65, [65, 64, 63, 1, 0], False),   # its blocks of 64 rows
    (200, 5, 6, 2, 64, 200, None, True),                # several units per CTA
    (150, 1, 8, 1, 256, 700, None, True),
    (160, 2, 4, 2, 128, 500, None, False),
    (150, 2, 1, 1, 64, 8300, None, True),               # more blocks than the sort has bins
    (40, 1, 3, 3, 64, 3000, None, True),                # cut units of more than 32 observations
    (20, 260, 4, 4, 64, 2600, None, True),              # cut, and more units than CTAs
    (40, 40, 8, 2, 256, 2400, None, True),
    (100, 17, 2, 2, 128, 2500, None, True),
]


def check(torch, st, layer, q, lens, pads, out, lse, scale=None):
    B, n_q, S, hd = q.shape
    seen = visible(torch, st.cap, lens, pads)
    z = scores(st, layer, q, scale).masked_fill(~seen[:, None, None], -math.inf)
    rl = torch.logsumexp(z, -1)
    p = torch.exp(z - rl[..., None].masked_fill((rl == -math.inf)[..., None], 0))
    v = st.v[layer].double().masked_fill(~seen[:, None, :, None], 0)
    ro, ra = p @ v, p @ v.abs()
    fold = lambda t: t.reshape(B, n_q, S, hd).transpose(1, 2).reshape(B, S, n_q * hd)
    fin = z.masked_fill(z == -math.inf, 0).abs().max().item()
    e = (hd ** 0.5 * (q.double().abs().amax() * 4.5 * hd ** 0.5 * (scale or hd ** -0.5)).item() + 4 * 1.45 * 2 * fin + 4) * 2.0 ** -24
    err = (out.double() - fold(ro)).abs()
    within = (err <= 2.0 ** -8 * fold(ro).abs() + (2.0 ** -8 + 2 * e + (st.cap + 128) * 2.0 ** -24) * fold(ra)).all().item()
    assert within, (err / fold(ra).clamp(min=1e-30)).max().item()
    rl = rl.reshape(B, n_q, S)
    none = rl == -math.inf
    assert torch.equal(none, lse == -math.inf)
    err = (lse.double() - rl).abs().masked_fill(none, 0)
    within = (err <= 2 * e + 2.0 ** -22 * (rl.abs().masked_fill(none, 0) + 1)).all().item()
    assert within, err.max().item()


@pytest.mark.gpu
@pytest.mark.parametrize("B,S,n_q,n_kv,hd,cap,lens,pad", CASES)
def test_against_the_formula(B, S, n_q, n_kv, hd, cap, lens, pad):
    torch = require_cuda()
    import vla_cpp_b200 as vb

    torch.manual_seed(B + S)
    st, q, lens, pads, g = make(torch, B, S, n_q, n_kv, hd, cap, lens, pad, seed=B * 100 + S)
    seen = visible(torch, cap, lens, pads)
    st.k[1].masked_fill_(~seen[:, None, :, None], math.nan)
    st.v[1].masked_fill_(~seen[:, None, :, None], math.inf)
    clean = vb.KvStore(2, B, n_kv, hd, cap, 0)
    clean.k.copy_(st.k.masked_fill(~seen[None, :, None, :, None], 0))
    clean.v.copy_(st.v.masked_fill(~seen[None, :, None, :, None], 0))
    results = []
    for split in (True, False):
        out = torch.full((B, S, n_q * hd), 77.0, dtype=torch.bfloat16, device="cuda")
        out, lse = vb.cross_attention(st, 1, q, lens=lens, pad_ranges=pads, out=out, split=split)
        assert vb.device_status() == 0
        check(torch, clean, 1, q, lens, pads, out, lse)
        results.append((out, lse))
        again = vb.cross_attention(st, 1, q, lens=lens, pad_ranges=pads, split=split)
        assert torch.equal(again[0], out) and torch.equal(again[1], lse)


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_growing_keys_rescale(hd):
    """Keys whose norm grows along the cache: the running maximum rises again and again, in both tiles and across pieces of a unit."""
    torch = require_cuda()
    import vla_cpp_b200 as vb

    st, q, lens, _, g = make(torch, 2, 40, 8, 1, hd, 1600, [1600, 1111], False, 3)
    st.k.mul_(torch.linspace(0.05, 6.0, 1600, device="cuda").bfloat16()[:, None])
    for split in (True, False):
        out, lse = vb.cross_attention(st, 0, q, lens=lens, split=split)
        check(torch, st, 0, q, lens, None, out, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_growing_keys_under_one_token(hd):
    """The same with few query rows: every block of 64 rows raises each warp's maximum."""
    torch = require_cuda()
    import vla_cpp_b200 as vb

    st, q, lens, pads, g = make(torch, 2, 1, 8, 2, hd, 1600, [1600, 1111], True, 6)
    st.k.mul_(torch.linspace(0.05, 6.0, 1600, device="cuda").bfloat16()[:, None])
    for split in (True, False):
        out, lse = vb.cross_attention(st, 0, q, lens=lens, pad_ranges=pads, split=split)
        assert vb.device_status() == 0
        check(torch, st, 0, q, lens, pads, out, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_lengths_by_default_and_out_of_range_and_a_scale(hd):
    torch = require_cuda()
    import vla_cpp_b200 as vb

    st, q, lens, _, g = make(torch, 3, 5, 4, 2, hd, 200, [150] * 3, False, 7)
    out, lse = vb.cross_attention(st, 0, q, max_len=150, scale=0.07)
    check(torch, st, 0, q, lens, None, out, lse, scale=0.07)
    odd = torch.tensor([-4, 2 ** 31 - 1, 150], dtype=torch.int32, device="cuda")
    o2, l2 = vb.cross_attention(st, 0, q, lens=odd, max_len=150, scale=0.07)
    check(torch, st, 0, q, torch.tensor([0, 150, 150], device="cuda"), None, o2, l2, scale=0.07)
    o3, l3 = vb.cross_attention(st, 0, q, max_len=0)
    assert not o3.any() and bool((l3 == -math.inf).all())


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 256])
def test_hidden_ranges_at_the_borders(hd):
    """Ranges that are empty, turned round, reach out of the rows on either side, or hide everything; lengths at the blocks' borders."""
    torch = require_cuda()
    import vla_cpp_b200 as vb

    lo_hi = [(0, 0), (9, 3), (-2 ** 31, 5), (250, 2 ** 31 - 1), (-2 ** 31, 2 ** 31 - 1), (0, 128), (128, 256), (127, 129), (-7, -3), (2 ** 31 - 1, 2 ** 31 - 1)]
    lens = [256, 255, 129, 256, 256, 128, 256, 129, 1, 127]
    B = len(lens)
    st, q, lens, _, g = make(torch, B, 3, 4, 2, hd, 256, lens, False, 17)
    pads = torch.tensor(lo_hi, dtype=torch.int32, device="cuda")
    out, lse = vb.cross_attention(st, 0, q, lens=lens, pad_ranges=pads)
    assert vb.device_status() == 0
    check(torch, st, 0, q, lens, pads.long(), out, lse)
    mass = vb.key_mass(st, 0, q, lse, lens=lens, pad_ranges=pads)
    seen = visible(torch, 256, lens, pads.long())
    z = scores(st, 0, q).masked_fill(~seen[:, None, None], -math.inf)
    want = torch.exp(z - lse.double().reshape(B, 2, -1, 1).nan_to_num(neginf=math.inf)).sum(2)
    torch.testing.assert_close(mass.double(), want, rtol=1e-4, atol=0)


@pytest.mark.gpu
def test_refusals():
    torch = require_cuda()
    import vla_cpp_b200 as vb

    st, q, lens, _, _ = make(torch, 2, 3, 4, 2, 64, 20, [20, 20], False, 7)
    z = lambda *s, t=torch.float32: torch.zeros(s, dtype=t, device="cuda")
    for kw in (dict(q=q.float()), dict(q=q.cpu()), dict(q=q[0]), dict(q=q.transpose(1, 2)), dict(q=q[:1]), dict(lens=z(2)), dict(lens=lens.cpu()),
               dict(pad_ranges=z(2, t=torch.int32)), dict(out=z(2, 3, 256)), dict(lse=z(2, 3, 4)), dict(max_len=21), dict(max_len=-1), dict(layer=2),
               dict(scale=-1.0), dict(out=q.view(2, 3, 256)), dict(q=z(2, 3, 3, 64, t=torch.bfloat16)), dict(q=z(2, 4, 0, 64, t=torch.bfloat16))):
        kw = {**dict(q=q, layer=0), **kw}
        with pytest.raises(vb.VlaB200Error) as e:
            vb.cross_attention(st, kw.pop("layer"), kw.pop("q"), **kw)
        assert e.value.code == -1, kw


def test_no_block_leaves_before_it_has_waited():
    """A block that ends without griddepcontrol.wait lets the next kernel take this one's end for the end of the one in front, whose results it
    may then read too early: no kernel that waits returns before it does."""
    import glob
    import os

    from tests.test_dependent_launch_sources import CSRC, functions, strip_comments

    waiting = 0
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu"))):
        for name, _, body in functions(strip_comments(open(path).read()), r"__global__"):
            if "pdl_wait" in body:
                waiting += 1
                assert "return;" not in body[:body.index("pdl_wait")], f"{os.path.basename(path)}: {name}"
    assert waiting > 20

"""kv_evict: rows, order, ties and what is left alone, exactly; and the cache it leaves, through the calls that read it."""
import ctypes as C
import math

import pytest

from tests.gpu_util import require_cuda


def test_argument_checks_need_no_gpu():
    from vla_cpp_b200 import api

    def call(**kw):
        def store(pre, base):
            g = lambda n, d: kw.pop(pre + n, d)
            return api._KvStoreC(g("k", base), g("v", base + 2 ** 20), g("layers", 1), g("obs", 2), g("n_kv", 1), g("hd", 64), g("cap", 8), 0)

        a, b = store("s_", 2 ** 24), store("d_", 2 ** 25)
        p = lambda n, d: C.c_void_p(kw.pop(n, d) or None)
        g = lambda n, d: kw.pop(n, d)
        return api.lib().vlab200_kv_evict(C.byref(a), C.byref(b), p("mass", 2 ** 26), p("lens", 2 ** 26 + 4096), g("max_len", 8), g("keep", 4),
                                          g("sink", 0), g("recent", 0), p("kept", 2 ** 27), p("mass_out", 2 ** 28), p("lens_out", 2 ** 29), None)

    for bad in (dict(s_k=None), dict(d_v=None), dict(mass=None), dict(kept=None), dict(s_layers=2), dict(s_obs=3), dict(d_n_kv=2), dict(d_hd=128),
                dict(max_len=9), dict(max_len=-1), dict(keep=0), dict(keep=9), dict(sink=-1), dict(recent=-1), dict(sink=3, recent=2),
                dict(sink=2 ** 31 - 1, recent=2), dict(s_k=2 ** 24 + 8), dict(d_k=2 ** 24), dict(d_k=2 ** 24 + 16), dict(d_v=2 ** 25 + 16),
                dict(mass_out=2 ** 26), dict(kept=2 ** 26 + 60), dict(lens_out=2 ** 26 + 4096), dict(lens_out=2 ** 28), dict(s_cap=0)):
        assert call(**bad) == -1, bad
    assert call(s_hd=80, d_hd=80) == -4


def chosen(w, n, keep, sink, recent):
    """Indices of the kept rows of one page, in order: plain Python."""
    def rank(i):
        if i < sink or i >= n - recent:
            return math.inf, 1
        return (-math.inf, -1) if math.isnan(w[i]) else (w[i], 0)

    return sorted(sorted(range(n), key=lambda i: (*(-x for x in rank(i)), i))[:keep])


CASES = [
    # L, B, n_kv, hd, cap, lens, keep, dst cap, sink, recent, weights
    (1, 1, 1, 64, 1, [1], 1, 1, 0, 0, "spread"),
    (2, 3, 2, 64, 241, [241, 0, 100], 100, 151, 1, 49, "spread"),
    (1, 2, 5, 128, 300, [300, 257], 256, 256, 0, 0, "few values"),
    (1, 2, 1, 256, 700, [700, 513], 1, 5, 0, 0, "spread"),
    (1, 2, 1, 64, 600, [600, 599], 598, 600, 300, 298, "spread"),   # protected rows fill the budget
    (1, 3, 2, 128, 40, [40, 3, 9], 8, 8, 4, 4, "zero"),             # and overlap in the short ones
    (3, 2, 1, 256, 900, [900, 899], 450, 500, 4, 48, "any"),        # infinities, no-numbers, negative and denormal weights
    (1, 4, 3, 64, 513, [512, 513, 511, 1], 257, 300, 0, 1, "exponents"),
    (2, 2, 1, 64, 1024, [1024, 993], 992, 1000, 2, 31, "few values"),
    (1, 3, 2, 64, 1025, [1025, 1024, 0], 1024, 1024, 0, 0, "any"),   # a block per page from here on
    (1, 2, 1, 128, 5000, [5000, 1300], 1299, 1300, 10, 200, "few values"),
    (1, 2, 2, 64, 3000, [3000, 2999], 100, 100, 0, 0, "any"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("L,B,n_kv,hd,cap,lens,keep,dcap,sink,recent,weights", CASES)
def test_rows_order_and_ties(L, B, n_kv, hd, cap, lens, keep, dcap, sink, recent, weights):
    torch = require_cuda()
    import vla_cpp_b200 as vb

    g = torch.Generator(device="cuda").manual_seed(keep)
    src, dst = vb.KvStore(L, B, n_kv, hd, cap, 0), vb.KvStore(L, B, n_kv, hd, dcap, 0)
    for t in (src.k, src.v, dst.k, dst.v):
        t.normal_(0, 1, generator=g)
    shape = (L, B, n_kv, cap)
    mass = torch.rand(shape, device="cuda", generator=g)
    if weights == "few values":
        mass = (mass * 4).floor() / 4 * (1 - 2 * (mass > 0.9).float())  # 0, -0, 1/4 ..: ties, both zeros
    if weights == "zero":
        mass.zero_()
    if weights == "exponents":
        mass = torch.exp2(torch.floor(mass * 250 - 125))
    if weights == "any":
        pick = torch.randint(0, 12, shape, device="cuda", generator=g)
        for i, x in enumerate((math.inf, -math.inf, math.nan, -math.nan, 1e-42, -1e-42, -3.0)):
            mass[pick == i] = x
    lens_t = torch.tensor(lens, dtype=torch.int32, device="cuda")
    k0, v0, src0 = dst.k.clone(), dst.v.clone(), (src.k.clone(), src.v.clone(), mass.clone())
    lens_out, kept, mass_out = vb.kv_evict(src, dst, mass, keep, lens=lens_t, sink=sink, recent=recent)
    assert vb.device_status() == 0
    assert lens_out.tolist() == [min(n, keep) for n in lens]
    w = mass.cpu()
    for l in range(L):
        for b in range(B):
            for h in range(n_kv):
                rows = chosen(w[l, b, h].tolist(), lens[b], keep, sink, recent)
                n = len(rows)
                assert kept[l, b, h].tolist() == rows + [-1] * (keep - n)
                at = torch.tensor(rows, dtype=torch.long, device="cuda")
                bits = lambda t: t.view(torch.int16)
                assert torch.equal(bits(dst.k[l, b, h, :n]), bits(src.k[l, b, h][at])) and torch.equal(bits(dst.v[l, b, h, :n]), bits(src.v[l, b, h][at]))
                assert torch.equal(dst.k[l, b, h, n:], k0[l, b, h, n:]) and torch.equal(dst.v[l, b, h, n:], v0[l, b, h, n:])
                assert torch.equal(mass_out[l, b, h, :n].view(torch.int32), mass[l, b, h][at].view(torch.int32)) and not mass_out[l, b, h, n:].any()
    assert torch.equal(src.k, src0[0]) and torch.equal(src.v, src0[1]) and torch.equal(mass.view(torch.int32), src0[2].view(torch.int32))


@pytest.mark.gpu
def test_lengths_by_default_and_out_of_range():
    torch = require_cuda()
    import vla_cpp_b200 as vb

    src, dst = vb.KvStore(1, 3, 1, 64, 50, 0), vb.KvStore(1, 3, 1, 64, 20, 0)
    src.k.normal_()
    mass = torch.rand(1, 3, 1, 50, device="cuda")
    lens, kept, _ = vb.kv_evict(src, dst, mass, 20, max_len=40)
    assert lens.tolist() == [20] * 3 and kept.max() < 40
    got = vb.kv_evict(src, dst, mass, 20, lens=torch.tensor([-5, 2 ** 31 - 1, 40], dtype=torch.int32, device="cuda"), max_len=40)
    assert got[0].tolist() == [0, 20, 20] and torch.equal(got[1][0, 1:], kept[0, 1:]) and (got[1][0, 0] == -1).all()
    assert vb.kv_evict(src, dst, mass, 20, max_len=0)[0].tolist() == [0] * 3


@pytest.mark.gpu
def test_refusals():
    torch = require_cuda()
    import vla_cpp_b200 as vb

    src, dst = vb.KvStore(1, 2, 1, 64, 50, 0), vb.KvStore(1, 2, 1, 64, 20, 0)
    mass = torch.rand(1, 2, 1, 50, device="cuda")
    z = lambda *s, t=torch.float32: torch.zeros(s, dtype=t, device="cuda")
    for kw in (dict(dst=src), dict(dst=vb.KvStore(2, 2, 1, 64, 20, 0)), dict(dst=vb.KvStore(1, 2, 1, 128, 20, 0)), dict(mass=mass.cpu()),
               dict(mass=mass[..., :49]), dict(mass=mass.double()), dict(keep=21), dict(keep=0), dict(sink=11, recent=10), dict(lens=z(2)),
               dict(kept=z(1, 2, 1, 19, t=torch.int32)), dict(mass_out=z(1, 2, 1, 50)), dict(lens_out=z(2, t=torch.int64)), dict(max_len=51)):
        kw = {**dict(dst=dst, mass=mass, keep=20), **kw}
        with pytest.raises(vb.VlaB200Error) as e:
            vb.kv_evict(src, kw.pop("dst"), kw.pop("mass"), kw.pop("keep"), **kw)
        assert e.value.code == -1, kw

"""key_mass against its formula in 64 bits.

Bound of an element, relative to its sum of weights W: the score's product and sum of head_dim terms in 32 bits (inputs are exact), at
most head_dim 2^-24 of sum |q_i k_i| scale <= Z; the exponent's scaling, subtraction and lse in powers of two, 4 x 2^-24 of its
magnitude E; the exponential (2^-22); the sum, 2^-24 x its depth (columns of a thread, <= rows / 2 + chunks) -- all of it relative to
each weight: (hd Z + 4 E + 4 + R / 2) 2^-24 W, and one rounding of decay * mass + W."""
import ctypes as C
import math

import pytest

from tests.gpu_util import require_cuda


def test_argument_checks_need_no_gpu():
    from vla_cpp_b200 import api

    def call(**kw):
        st = api._KvStoreC(*(kw.pop(n, d) for n, d in (("k", 1 << 20), ("v", 2 << 20), ("layers", 1), ("obs", 2), ("n_kv", 1), ("hd", 64),
                                                       ("cap", 8), ("prefix", 0))))
        g = lambda n, d: kw.pop(n, d)
        p = lambda v: C.c_void_p(v) if v else None
        return api.lib().vlab200_key_mass(C.byref(st), g("layer", 0), p(g("q", 3 << 20)), p(g("lse", 4 << 20)), p(g("mass", 5 << 20)), p(g("out", 6 << 20)),
                                          g("S", 1), g("n_q", 2), None, g("max_len", 0), None, C.c_float(g("scale", 0.0)),
                                          C.c_float(g("decay", 1.0)), None)

    assert call() == 0  # no rows
    for bad in (dict(k=None), dict(q=None), dict(lse=None), dict(out=None), dict(layer=1), dict(layer=-1), dict(S=0), dict(n_q=0),
                dict(n_q=3, n_kv=2), dict(max_len=9), dict(max_len=-1), dict(scale=-1.0), dict(scale=math.nan), dict(decay=-0.5),
                dict(decay=math.nan), dict(q=24), dict(k=8), dict(max_len=8, out=3 << 20), dict(max_len=8, out=4 << 20), dict(max_len=8, out=1 << 20),
                dict(max_len=8, out=(5 << 20) + 4)):
        assert call(**bad) == -1, bad
    assert call(hd=80) == -4


CASES = [
    # B, S, n_q, n_kv, hd, cap, lens, pad, decay
    (1, 1, 8, 1, 256, 1, [1], False, 1.0),
    (1, 1, 20, 5, 128, 1001, [1001], False, 0.5),
    (2, 1, 1, 1, 64, 130, [129, 128], False, 1.0),
    (4, 50, 15, 5, 64, 241, [241, 0, 113, 127], True, 0.5),
    (3, 51, 8, 1, 256, 300, [300, 1, 257], True, 0.0),
    (2, 17, 4, 4, 128, 260, [5, 260], False, 0.25),       # 17 rows per item: one over the column block of 16
    (2, 33, 2, 1, 64, 140, [140, 64], False, 1.0),        # 66 rows: two columns into the second half
    (1, 129, 3, 1, 128, 390, [385], True, 1.0),           # 387 rows: four chunks, the last of three rows
    (40, 3, 6, 2, 64, 700, None, False, 1.0),             # more units than CTAs
    (30, 20, 4, 2, 128, 900, None, True, 0.5),
    (9, 16, 8, 2, 256, 1100, None, False, 0.5),
]


def make(torch, B, S, n_q, n_kv, hd, cap, lens, pad, seed, layers=2):
    import vla_cpp_b200 as vb

    g = torch.Generator(device="cuda").manual_seed(seed)
    st = vb.KvStore(layers, B, n_kv, hd, cap, 0)
    st.k.normal_(0, 1, generator=g)
    st.v.normal_(0, 1, generator=g)
    q = (torch.randn(B, n_q, S, hd, device="cuda", generator=g) * 1.5).bfloat16()
    lens = torch.tensor(lens, dtype=torch.int32) if lens is not None else torch.randint(0, cap + 1, (B,), dtype=torch.int32)
    pads = None
    if pad:
        lo = (lens * torch.rand(B)).int()
        pads = torch.stack((lo, torch.minimum(lo + 1 + (lens * 0.4 * torch.rand(B)).int(), lens)), 1).int().cuda().contiguous()
    return st, q, lens.cuda(), pads, g


def visible(torch, cap, lens, pads):
    at = torch.arange(cap, device="cuda")
    seen = at[None] < lens[:, None]
    if pads is not None:
        seen &= (at[None] < pads[:, :1]) | (at[None] >= pads[:, 1:])
    return seen


def scores(st, layer, q, scale=None):
    """float64 [B, n_kv, g * S, cap]."""
    B, n_q, S, hd = q.shape
    return q.double().reshape(B, st.n_kv, -1, hd) @ st.k[layer].double().transpose(-1, -2) * (scale or hd ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("B,S,n_q,n_kv,hd,cap,lens,pad,decay", CASES)
def test_against_the_formula(B, S, n_q, n_kv, hd, cap, lens, pad, decay):
    torch = require_cuda()
    import vla_cpp_b200 as vb

    torch.manual_seed(B + S)
    st, q, lens, pads, g = make(torch, B, S, n_q, n_kv, hd, cap, lens, pad, seed=B * 100 + S)
    seen = visible(torch, cap, lens, pads)
    z = scores(st, 1, q).masked_fill(~seen[:, None, None], -math.inf)
    lse = torch.logsumexp(z, -1).float()
    rel = (z - lse.double()[..., None]).masked_fill((lse == -math.inf)[..., None], -math.inf)
    w = torch.exp(rel).sum(2)
    mass = torch.rand(B, n_kv, cap, device="cuda", generator=g)
    before = torch.full((B, n_kv, cap), 5.0, device="cuda")
    # what is behind an observation's rows, and what is hidden, may be anything
    st.k[1].masked_fill_(~seen[:, None, :, None], math.nan)
    out = vb.key_mass(st, 1, q, lse.reshape(B, n_q, S), lens=lens, pad_ranges=pads, decay=decay, mass=mass, out=before.clone())
    assert vb.device_status() == 0
    live = (torch.arange(cap, device="cuda")[None] < lens[:, None])[:, None].expand_as(out)
    want = torch.where(live, decay * mass.double() + w, before.double())
    Z = (q.double().abs().amax() * 3 * hd ** 0.5).item()
    E = (rel.masked_fill(rel == -math.inf, 0).abs().max() + lse[lse > -math.inf].abs().max()).item() * 1.45 if bool((lse > -math.inf).any()) else 0
    tol = (hd ** 0.5 * Z + 4 * E + 4 + n_q // n_kv * S / 2) * 2.0 ** -24 * w + want.abs() * 2.0 ** -23
    assert bool(((out.double() - want).abs() <= tol * live).all()), ((out.double() - want).abs() / want.abs().clamp(min=1e-30)).max().item()
    # in place, from nothing, and twice the same bits
    assert torch.equal(vb.key_mass(st, 1, q, lse.reshape(B, n_q, S), lens=lens, pad_ranges=pads, decay=decay, mass=mass, out=before.clone()), out)
    inplace = mass.clone()
    vb.key_mass(st, 1, q, lse.reshape(B, n_q, S), lens=lens, pad_ranges=pads, decay=decay, mass=inplace, out=inplace)
    assert torch.equal(inplace, torch.where(live, out, mass))
    fresh = vb.key_mass(st, 1, q, lse.reshape(B, n_q, S), lens=lens, pad_ranges=pads)
    assert bool(((fresh.double() - w * live).abs() <= tol).all())


@pytest.mark.gpu
def test_lengths_by_default_and_out_of_range_and_a_scale():
    torch = require_cuda()
    import vla_cpp_b200 as vb

    st, q, _, _, g = make(torch, 3, 2, 4, 2, 64, 200, [200] * 3, False, 7)
    z = scores(st, 0, q, 0.3)[..., :150]
    lse = torch.logsumexp(z, -1)
    want = torch.exp(z - lse[..., None]).sum(2)
    lse = lse.float().reshape(3, 4, 2)
    out = vb.key_mass(st, 0, q, lse, max_len=150, scale=0.3)
    torch.testing.assert_close(out[..., :150].double(), want, rtol=2e-5, atol=0)
    assert not out[..., 150:].any()
    lens = torch.tensor([-4, 2 ** 31 - 1, 150], dtype=torch.int32, device="cuda")
    got = vb.key_mass(st, 0, q, lse, lens=lens, max_len=150, scale=0.3)
    assert not got[0].any() and torch.equal(got[1:], out[1:])


@pytest.mark.gpu
def test_refusals():
    torch = require_cuda()
    import vla_cpp_b200 as vb

    st, q, lens, _, _ = make(torch, 2, 3, 4, 2, 64, 20, [20, 20], False, 7)
    lse = torch.zeros(2, 4, 3, device="cuda")
    z = lambda *s, t=torch.float32: torch.zeros(s, dtype=t, device="cuda")
    for kw in (dict(out=lse.new_zeros(1).expand(80).reshape(2, 2, 20)[:1]), dict(q=q.float()), dict(q=q.cpu()), dict(q=q[0]), dict(q=q.transpose(1, 2)), dict(q=q[:1]), dict(lse=lse.half()), dict(lse=z(2, 3, 4)),
               dict(lens=z(2)), dict(lens=z(3, t=torch.int32)), dict(pad_ranges=z(2, t=torch.int32)), dict(mass=z(2, 2, 19)),
               dict(out=z(2, 2, 20, t=torch.bfloat16)), dict(max_len=21), dict(max_len=-1), dict(layer=2), dict(decay=-1.0),
               dict(q=z(2, 3, 3, 64, t=torch.bfloat16), lse=z(2, 3, 3))):
        kw = {**dict(q=q, lse=lse, layer=0, lens=lens), **kw}
        with pytest.raises(vb.VlaB200Error) as e:
            vb.key_mass(st, kw.pop("layer"), kw.pop("q"), kw.pop("lse"), **kw)
        assert e.value.code == -1, kw
    both = z(2 * 2 * 20 + 4)  # weights that overlap the ones they replace without being them
    with pytest.raises(vb.VlaB200Error):
        vb.key_mass(st, 0, q, lse, lens=lens, mass=both[:80].view(2, 2, 20), out=both[4:].view(2, 2, 20))

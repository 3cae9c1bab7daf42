"""qk_norm_rope_append and rope_freqs against their formulas in 64 bits.

Bound of a q or k element: half a bf16 step of the value (2^-8 relative) plus what 32 bits lose in front of it, relative to the
rotated pair's magnitude A = m (|y_u| + |y_v|): norm (13 additions of squares, halved by the root, root, quotient, product:
10 x 2^-24), rotation (3 x 2^-24), cosine and sine (3 x 2^-24), the angle's rounding to 32 bits after whole turns are gone
(2 pi x 2^-25) and, at positions up to 2^31, its product in 64 bits (5e-7): below 2e-6 A in all.  V is one rounding."""
import ctypes as C
import math

import numpy as np
import pytest

from tests.gpu_util import require_cuda


def freqs_ref(rot, base, scaling, factor, original):
    """The published forms, pair by pair."""
    out = []
    for i in range(rot // 2):
        b = base * factor ** (rot / (rot - 2)) if scaling == "ntk" and rot > 2 else base
        f = 1.0 / b ** (2 * i / rot)
        if scaling == "linear":
            f = f / factor
        if scaling == "yarn":
            lo = max(math.floor(rot * math.log(original / (32 * 2 * math.pi)) / (2 * math.log(base))), 0)
            hi = min(math.ceil(rot * math.log(original / (2 * math.pi)) / (2 * math.log(base))), rot - 1)
            keep = 1 - min(max((i - lo) / max(hi - lo, 0.001), 0), 1)
            f = f / factor * (1 - keep) + f * keep
        out.append(f)
    return np.array(out)


@pytest.mark.parametrize("rot,base,scaling,factor,original", [
    (64, 10000.0, "none", 1.0, 0), (128, 10000.0, "linear", 4.0, 0), (2, 10000.0, "ntk", 8.0, 0), (96, 500000.0, "ntk", 8.0, 0),
    (128, 10000.0, "yarn", 16.0, 4096), (64, 1000000.0, "yarn", 1.0, 32768), (18, 10000.0, "yarn", 40.0, 3)])
def test_rope_freqs(rot, base, scaling, factor, original):
    import vla_cpp_b200 as vb

    f, m = vb.rope_freqs(rot, base, scaling, factor, original, device="cpu")
    # a power's exponent is rounded once: 2^-53 x |ln f| < 14, and a handful of roundings around it
    np.testing.assert_allclose(f.numpy(), freqs_ref(rot, base, scaling, factor, original), rtol=32 * 2.0 ** -53)
    assert abs(m - (0.1 * math.log(factor) + 1.0 if scaling == "yarn" else 1.0)) <= 2.0 ** -23


def test_rope_freqs_refusals():
    import vla_cpp_b200 as vb

    for bad in (dict(rot_dim=3), dict(rot_dim=0), dict(rot_dim=-2), dict(rot_dim=8, scaling="other"), dict(rot_dim=8, base=1.0),
                dict(rot_dim=8, base=float("nan")), dict(rot_dim=8, scaling="linear", factor=0.5),
                dict(rot_dim=8, scaling="ntk", factor=float("inf")), dict(rot_dim=8, scaling="yarn", factor=2.0)):
        with pytest.raises(vb.VlaB200Error) as e:
            vb.rope_freqs(device="cpu", **bad)
        assert e.value.code == -1, bad


def test_argument_checks_need_no_gpu():
    from vla_cpp_b200 import api

    def call(**kw):
        st = api._KvStoreC(*(kw.pop(n, d) for n, d in (("k", 16), ("v", 16), ("layers", 1), ("obs", 2), ("n_kv", 1), ("hd", 64),
                                                       ("cap", 8), ("prefix", 0))))
        layer = kw.pop("layer", 0)
        d = dict(x=16, x_stride=256, freqs=16, q_out=16, S=0, n_q=2, rot_dim=64, with_kv=1, eps=1e-6, mscale=1.0)
        d.update(kw)
        return api.lib().vlab200_qk_norm_rope_append(C.byref(st), layer, C.byref(api._QkNormRopeArgs(**d)), None)

    assert call() == 0  # no tokens
    for bad in (dict(x=None), dict(q_out=None), dict(k=None), dict(freqs=None), dict(layer=1), dict(layer=-1), dict(S=-1), dict(n_q=0),
                dict(x_stride=255), dict(x_stride=260), dict(x=24), dict(q_out=8), dict(rot_dim=66), dict(rot_dim=3), dict(rot_dim=-2),
                dict(eps=-1.0), dict(eps=float("nan")), dict(cap=0)):
        assert call(**bad) == -1, bad
    assert call(hd=80, x_stride=400) == -4
    assert call(with_kv=0, k=None, v=None, x_stride=128) == 0
    assert call(rot_dim=0, freqs=None) == 0


def reference(x, n_q, n_kv, hd, B, S, f, mscale, wq, wk, eps, inter, pos, with_kv):
    """-> q, k, v float64 [B, S, heads, hd] and the bound of every q and k element in front of its rounding."""
    import torch

    rot = 2 * len(f)
    x = x[:, :(n_q + (2 * n_kv if with_kv else 0)) * hd].double().reshape(B, S, -1, hd)
    ang = pos.double()[..., None] * torch.tensor(f, dtype=torch.float64, device=x.device)
    c, s = torch.cos(ang)[:, :, None] * mscale, torch.sin(ang)[:, :, None] * mscale
    iu = torch.arange(rot // 2, device=x.device) * (2 if inter else 1)
    iv = iu + (1 if inter else rot // 2)

    def part(h, w):
        if w is not None:
            h = h / torch.sqrt(h.square().mean(-1, keepdim=True) + eps) * w.double()
        out, amp = h.clone(), h.abs()
        u, v = h[..., iu], h[..., iv]
        out[..., iu], out[..., iv] = u * c - v * s, v * c + u * s
        amp[..., iu] = amp[..., iv] = mscale * (u.abs() + v.abs())
        return out, amp

    q, aq = part(x[:, :, :n_q], wq)
    if not with_kv:
        return q, aq, None, None, None
    k, ak = part(x[:, :, n_q:n_q + n_kv], wk)
    return q, aq, k, ak, x[:, :, n_q + n_kv:]


def check(got, ref, amp):
    err = (got.double() - ref).abs() - ref.abs() * 2.0 ** -8 * (1 + 2.0 ** -15) - 2e-6 * amp
    assert bool((err <= 0).all()), err.max().item()


CASES = [
    # B, S, n_q, n_kv, hd, rot, inter, f32, norms, ragged, pos0, scaling
    (1, 1, 8, 1, 256, 256, False, False, "qk", False, 0, "none"),
    (1, 1, 20, 5, 128, 128, False, False, "qk", False, 2 ** 31 - 2, "yarn"),
    (3, 7, 15, 5, 64, 32, True, True, "qk", True, 1000003, "none"),
    (2, 51, 15, 5, 64, 64, False, False, "q", False, 241, "linear"),
    (5, 33, 3, 1, 64, 20, False, False, "qk", True, 77, "ntk"),     # partners in the middle of a lane's columns
    (2, 19, 4, 4, 128, 2, True, False, "k", False, 5, "none"),
    (2, 19, 1, 1, 128, 126, False, True, "", True, 90000, "yarn"),
    (1, 130, 2, 2, 256, 0, False, False, "qk", False, 0, "none"),  # norms alone
    (4, 700, 5, 1, 256, 128, False, False, "qk", True, 10, "none"),  # more tokens than warps
    (130, 1, 7, 7, 64, 16, False, True, "qk", False, 3, "none"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("B,S,n_q,n_kv,hd,rot,inter,f32,norms,ragged,pos0,scaling", CASES)
def test_against_the_formula(B, S, n_q, n_kv, hd, rot, inter, f32, norms, ragged, pos0, scaling):
    torch = require_cuda()
    import vla_cpp_b200 as vb

    g = torch.Generator(device="cuda").manual_seed(B * 1000 + S)
    width = (n_q + 2 * n_kv) * hd
    for with_kv in (True, False):
        for shift in (0, 8):  # columns in front of the first head, and behind the last
            w = (width if with_kv else n_q * hd)
            big = torch.randn(B * S, w + 2 * shift, device="cuda", generator=g) * 2
            big = big if f32 else big.bfloat16()
            x = big[:, shift:shift + w]
            wq = 1 + 0.2 * torch.randn(hd, device="cuda", generator=g) if "q" in norms else None
            wk = 1 + 0.2 * torch.randn(hd, device="cuda", generator=g) if "k" in norms else None
            freqs, m = vb.rope_freqs(rot, 10000.0, scaling, 8.0, 4096) if rot else (None, 1.0)
            f = freqs_ref(rot, 10000.0, scaling, 8.0, 4096)
            pos = torch.randint(max(pos0 - 99, 0), pos0 + 1, (B, S), device="cuda", generator=g, dtype=torch.int32)
            row0 = torch.randint(0, 6, (B,), device="cuda", generator=g, dtype=torch.int32)
            n_tok = torch.randint(0, S + 1, (B,), device="cuda", generator=g, dtype=torch.int32) if ragged else None
            st = vb.KvStore(2, B, n_kv, hd, 3, S + 3)
            st.k.fill_(7.0)
            st.v.fill_(9.0)
            q = vb.qk_norm_rope_append(st, 1, x, S, n_q, freqs, wq, wk, eps=1e-6, interleaved=inter, mscale=m, pos=pos, row0=row0,
                                       n_tok=n_tok, with_kv=with_kv)
            assert vb.device_status() == 0
            rq, aq, rk, ak, rv = reference(x, n_q, n_kv, hd, B, S, f, m, wq, wk, 1e-6, inter, pos, with_kv)
            live = torch.arange(S, device="cuda")[None] < (n_tok[:, None] if ragged else S)
            mask = live[:, :, None, None]
            check(q.transpose(1, 2), rq * mask, aq)
            assert not q.transpose(1, 2).masked_select(~mask).any()
            rest_k, rest_v = torch.ones_like(st.k[1], dtype=torch.bool), None
            for b in range(B) if with_kv else ():
                n = int(n_tok[b]) if ragged else S
                r = int(row0[b])
                check(st.k[1, b, :, r:r + n].transpose(0, 1), rk[b, :n], ak[b, :n])
                assert torch.equal(st.v[1, b, :, r:r + n].transpose(0, 1), rv[b, :n].to(torch.bfloat16))
                rest_k[b, :, r:r + n] = False
            assert (st.k[1].masked_select(rest_k) == 7.0).all() and (st.v[1].masked_select(rest_k) == 9.0).all()
            assert (st.k[0] == 7.0).all() and (st.v[0] == 9.0).all()


@pytest.mark.gpu
def test_rows_and_positions_by_default_and_at_the_borders():
    """Without row0 the rows start at prefix_len, without pos a token's position is its row; rows outside the page are left out."""
    torch = require_cuda()
    import vla_cpp_b200 as vb

    g = torch.Generator(device="cuda").manual_seed(3)
    B, S, n_q, n_kv, hd, P = 3, 4, 2, 1, 64, 10
    x = torch.randn(B * S, (n_q + 2 * n_kv) * hd, device="cuda", generator=g).bfloat16()
    freqs, m = vb.rope_freqs(hd)
    f = freqs_ref(hd, 10000.0, "none", 1.0, 0)
    st = vb.KvStore(1, B, n_kv, hd, P, S)
    q = vb.qk_norm_rope_append(st, 0, x, S, n_q, freqs)
    pos = torch.arange(P, P + S, device="cuda", dtype=torch.int32).expand(B, S)
    rq, aq, rk, ak, rv = reference(x, n_q, n_kv, hd, B, S, f, 1.0, None, None, 0.0, False, pos, True)
    check(q.transpose(1, 2), rq, aq)
    check(st.k[0, :, :, P:].transpose(1, 2), rk, ak)
    assert not st.k[0, :, :, :P].any()
    row0 = torch.tensor([-2, 2 ** 31 - 3, P + 2], dtype=torch.int32, device="cuda")
    st2 = vb.KvStore(1, B, n_kv, hd, P, S)
    n = torch.tensor([S, S, S + 100], dtype=torch.int32, device="cuda")
    q2 = vb.qk_norm_rope_append(st2, 0, x, S, n_q, freqs, pos=pos.contiguous(), row0=row0, n_tok=n)
    assert torch.equal(q2, q)
    want = torch.zeros_like(st.v[0]).float()
    want[0, :, :2] = rv[0, 2:].transpose(0, 1)
    want[2, :, P + 2:] = rv[2, :2].transpose(0, 1)
    assert torch.equal(st2.v[0].float(), want)


@pytest.mark.gpu
def test_refusals():
    torch = require_cuda()
    import vla_cpp_b200 as vb

    B, S, n_q, hd = 2, 3, 2, 64
    st = vb.KvStore(1, B, 1, hd, 4, S)
    freqs, _ = vb.rope_freqs(hd)
    good = dict(x=torch.zeros(B * S, 4 * hd, dtype=torch.bfloat16, device="cuda"), S=S, n_q=n_q, freqs=freqs)
    z = lambda *s, t=torch.int32: torch.zeros(s, dtype=t, device="cuda")
    bad = [dict(x=good["x"].cpu()), dict(x=good["x"].half()), dict(x=good["x"][:, 1:]), dict(x=good["x"][:-1]), dict(x=good["x"].T),
           dict(S=S + 1), dict(n_q=3), dict(freqs=freqs.float()), dict(freqs=freqs.cpu()), dict(freqs=z(hd // 2 + 1, t=torch.float64)),
           dict(q_norm=z(hd + 1, t=torch.float32)), dict(k_norm=z(hd, t=torch.bfloat16)), dict(pos=z(B * S)), dict(row0=z(B, t=torch.int64)),
           dict(n_tok=z(B + 1)), dict(q_out=z(B, n_q, S, hd, t=torch.float32)), dict(q_out=z(B, S, n_q, hd, t=torch.bfloat16)),
           dict(layer=1), dict(eps=-1.0), dict(q_out=good["x"].view(-1)[:B * n_q * S * hd].view(B, n_q, S, hd))]
    for kw in bad:
        kw = {**good, "layer": 0, **kw}
        with pytest.raises(vb.VlaB200Error) as e:
            vb.qk_norm_rope_append(st, kw.pop("layer"), kw.pop("x"), kw.pop("S"), kw.pop("n_q"), **kw)
        assert e.value.code == -1, kw


@pytest.mark.gpu
def test_captured_and_replayed_and_on_another_stream():
    torch = require_cuda()
    import vla_cpp_b200 as vb

    g = torch.Generator(device="cuda").manual_seed(4)
    B, S, n_q, n_kv, hd = 4, 9, 4, 2, 128
    xs = [torch.randn(B * S, (n_q + 2 * n_kv) * hd, device="cuda", generator=g).bfloat16() for _ in range(2)]
    freqs, m = vb.rope_freqs(hd)
    want = []
    for x in xs:
        st = vb.KvStore(1, B, n_kv, hd, 5, S)
        want.append((vb.qk_norm_rope_append(st, 0, x, S, n_q, freqs), st.k, st.v))
    x, st = xs[0].clone(), vb.KvStore(1, B, n_kv, hd, 5, S)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        q = vb.qk_norm_rope_append(st, 0, x, S, n_q, freqs)
    side.synchronize()
    assert torch.equal(q, want[0][0]) and torch.equal(st.k, want[0][1]) and torch.equal(st.v, want[0][2])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = vb.qk_norm_rope_append(st, 0, x, S, n_q, freqs)
    for i in (1, 0, 1):
        x.copy_(xs[i])
        graph.replay()
        assert torch.equal(q, want[i][0]) and torch.equal(st.k, want[i][1]) and torch.equal(st.v, want[i][2])

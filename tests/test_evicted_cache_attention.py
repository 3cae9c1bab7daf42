"""vlab200_attention over a store that kv_evict filled, where every observation has at least as many rows as are kept: against the formula over the
rows that stayed.  Bound of an element: one bf16 rounding of the value, one of each weight (2^-8 each); what is done in 32 bits: a score's
sum is off by at most hd 2^-24 sum |q k| scale <= 256 x 2^-24 x 30 < 2^-11, in a weight and in the row's sum: 2^-10 of the weighted |v|."""
import pytest

from tests.gpu_util import require_cuda
from tests.test_cross_attention import check as check_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,P,S,n_q,n_kv,hd,keep", [(5, 150, 20, 6, 2, 64, 64), (3, 300, 9, 8, 1, 256, 100), (4, 200, 33, 4, 4, 128, 90), (2, 1400, 51, 8, 1, 256, 700)])
def test_attention_over_what_was_kept(B, P, S, n_q, n_kv, hd, keep):
    torch = require_cuda()
    import vla_cpp_b200 as vb

    g = torch.Generator(device="cuda").manual_seed(keep)
    st, small = vb.KvStore(1, B, n_kv, hd, 0, P), vb.KvStore(1, B, n_kv, hd, keep, S)
    st.k.normal_(0, 1, generator=g)
    st.v.normal_(0, 1, generator=g)
    lens = torch.randint(keep, P + 1, (B,), device="cuda", generator=g, dtype=torch.int32)
    lens[0], lens[-1] = keep, P
    q = torch.randn(B, n_q, S, hd, device="cuda", generator=g).bfloat16()
    _, lse = vb.cross_attention(st, 0, q, lens=lens)
    mass = vb.key_mass(st, 0, q, lse, lens=lens)
    left, kept, _ = vb.kv_evict(st, small, mass[None], keep, lens=lens, sink=2, recent=8)
    assert left.tolist() == [keep] * B
    at = kept[0].long()[..., None].expand(B, n_kv, keep, hd)
    k, v = st.k[0].gather(2, at), st.v[0].gather(2, at)
    assert torch.equal(small.k[0, :, :, :keep], k) and torch.equal(small.v[0, :, :, :keep], v)
    p = torch.softmax(q.double().reshape(B, n_kv, -1, hd) @ k.double().transpose(-1, -2) * hd ** -0.5, -1)
    fold = lambda t: t.reshape(B, n_q, S, hd).transpose(1, 2).reshape(B, S, n_q * hd)
    want, size = fold(p @ v.double()), fold(p @ v.double().abs())
    y = vb.attention(small, 0, q, S, n_q, keep, vb.MASK_NONE)
    assert vb.device_status() == 0
    err = (y.double() - want).abs()
    assert bool((err <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -10) * size).all()), (err / size).max().item()
    z, lse = vb.cross_attention(small, 0, q, lens=left)
    check_attention(torch, small, 0, q, left, None, z, lse)


@pytest.mark.parametrize("hd,n_q,n_kv,S", [(64, 6, 2, 20), (256, 8, 1, 1)])
def test_hidden_rows_go_where_enough_others_weigh_something(hd, n_q, n_kv, S):
    """Hidden rows weigh nothing: with no more rows kept than are visible, and none of the protected ones hidden, none of them is left."""
    torch = require_cuda()
    import vla_cpp_b200 as vb

    B, P, keep = 4, 180, 100
    g = torch.Generator(device="cuda").manual_seed(hd)
    st, small = vb.KvStore(1, B, n_kv, hd, 0, P), vb.KvStore(1, B, n_kv, hd, keep, 0)
    st.k.normal_(0, 1, generator=g)
    st.v.normal_(0, 1, generator=g)
    lens = torch.tensor([P, 150, 170, 130], dtype=torch.int32, device="cuda")
    pads = torch.tensor([[60, 100], [4, 54], [120, 130], [50, 80]], dtype=torch.int32, device="cuda")  # 140, 100, 160 and 100 visible rows
    for b, (lo, hi) in enumerate(pads.tolist()):
        st.k[:, b, :, lo:hi] = float("nan")
        st.v[:, b, :, lo:hi] = float("nan")
    q = torch.randn(B, n_q, S, hd, device="cuda", generator=g).bfloat16()
    _, lse = vb.cross_attention(st, 0, q, lens=lens, pad_ranges=pads)
    mass = vb.key_mass(st, 0, q, lse, lens=lens, pad_ranges=pads)
    left, kept, _ = vb.kv_evict(st, small, mass[None], keep, lens=lens, sink=4, recent=8)
    rows = kept[0].long()
    assert left.tolist() == [keep] * B
    assert not ((rows >= pads[:, None, :1]) & (rows < pads[:, None, 1:])).any()
    out, lse = vb.cross_attention(small, 0, q, lens=left)
    check_attention(torch, small, 0, q, left, None, out, lse)
    assert vb.device_status() == 0

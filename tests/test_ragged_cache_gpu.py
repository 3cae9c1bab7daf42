"""The operators of a ragged prefix cache as they are used together: rows in by qk_norm_rope_append, read by cross_attention, weighed by key_mass,
shrunk by kv_evict, read again -- there by the calls that know one prefix length too.  Every step is compared with the formula on the step's
own inputs, so a bound of one step does not have to hold through the others.  Captured, replayed and side by side on streams."""
import math

import pytest

from tests.gpu_util import require_cuda
from tests.test_cross_attention import check as check_attention
from tests.test_kv_evict import chosen
from tests.test_qk_norm_rope import check as check_rope, freqs_ref, reference

pytestmark = pytest.mark.gpu


def prompts(torch, B, P, n_q, n_kv, hd, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(B * P, (n_q + 2 * n_kv) * hd, device="cuda", generator=g).bfloat16()
    w = [1 + 0.1 * torch.randn(hd, device="cuda", generator=g) for _ in range(2)]
    lens = torch.randint(P // 3, P + 1, (B,), device="cuda", generator=g, dtype=torch.int32)
    lens[B // 2] = 0
    return x, w, lens, g


@pytest.mark.parametrize("B,P,S,n_q,n_kv,hd,keep", [(5, 150, 20, 6, 2, 64, 64), (3, 300, 9, 8, 1, 256, 100), (4, 200, 33, 4, 4, 128, 90)])
def test_fill_read_weigh_evict_read(B, P, S, n_q, n_kv, hd, keep):
    torch = require_cuda()
    import vla_cpp_b200 as vb

    x, (wq, wk), lens, g = prompts(torch, B, P, n_q, n_kv, hd, 11)
    freqs, m = vb.rope_freqs(hd, 10000.0, "yarn", 4.0, 128)
    st = vb.KvStore(1, B, n_kv, hd, 0, P + S)
    st.k.fill_(math.nan)  # rows that nobody wrote
    st.v.fill_(math.nan)
    row0 = torch.zeros(B, dtype=torch.int32, device="cuda")
    # the prompt: K / V of every live token
    qp = vb.qk_norm_rope_append(st, 0, x, P, n_q, freqs, wq, wk, mscale=m, row0=row0, n_tok=lens)
    pos = torch.arange(P, device="cuda", dtype=torch.int32).expand(B, P)
    rq, aq, rk, ak, rv = reference(x, n_q, n_kv, hd, B, P, freqs_ref(hd, 10000.0, "yarn", 4.0, 128), m, wq, wk, 1e-6, False, pos, True)
    for b, n in enumerate(lens.tolist()):
        check_rope(qp[b, :, :n].transpose(0, 1), rq[b, :n], aq[b, :n])
        check_rope(st.k[0, b, :, :n].transpose(0, 1), rk[b, :n], ak[b, :n])
        assert torch.equal(st.v[0, b, :, :n].transpose(0, 1), rv[b, :n].bfloat16()) and bool(st.k[0, b, :, n:].isnan().all())
    # query tokens on top of it, at the positions behind each observation's own prompt
    xs = torch.randn(B * S, n_q * hd, device="cuda", generator=g).bfloat16()
    at = (lens[:, None] + torch.arange(S, device="cuda", dtype=torch.int32)).contiguous()
    q = vb.qk_norm_rope_append(st, 0, xs, S, n_q, freqs, wq, mscale=m, pos=at, with_kv=False)
    out, lse = vb.cross_attention(st, 0, q, lens=lens)
    clean = vb.KvStore(1, B, n_kv, hd, 0, P + S)
    clean.k.copy_(st.k.nan_to_num(0.0))
    clean.v.copy_(st.v.nan_to_num(0.0))
    check_attention(torch, clean, 0, q, lens, None, out, lse)
    # what each row got; a page's weights add up to one per query row
    mass = vb.key_mass(st, 0, q, lse, lens=lens)
    total = mass.sum(-1)
    want = torch.where(lens > 0, n_q // n_kv * S, 0)[:, None].expand_as(total)
    torch.testing.assert_close(total, want.float(), rtol=1e-4, atol=0)
    # half of it goes
    small = vb.KvStore(1, B, n_kv, hd, keep, S)
    left, kept, _ = vb.kv_evict(st, small, mass[None], keep, lens=lens, sink=2, recent=8)
    assert vb.device_status() == 0
    w = mass.cpu()
    for b, n in enumerate(lens.tolist()):
        for h in range(n_kv):
            rows = chosen(w[b, h].tolist(), n, keep, 2, 8)
            assert kept[0, b, h].tolist() == rows + [-1] * (keep - len(rows))
    # what is left is read as before ...
    out2, lse2 = vb.cross_attention(small, 0, q, lens=left)
    check_attention(torch, small, 0, q, left, None, out2, lse2)
    # ... and where every observation keeps as many rows, by the call that has one length for all, after the action tokens' own rows
    if int(left[left > 0].min()) == keep:
        ones = torch.full((B,), keep, dtype=torch.int32, device="cuda")
        y = vb.attention(small, 0, q, S, n_q, keep, vb.MASK_NONE)
        z, _ = vb.cross_attention(small, 0, q, lens=ones)
        live = left > 0
        # each within (2^-8 + 2^-8) of its weighted |v|, which the largest |v| bounds
        assert ((y[live].float() - z[live].float()).abs().max() <= 2 * 2.0 ** -7 * small.v.float().abs().max()).item()


def test_captured_replayed_and_on_two_streams():
    """Two graphs of the same calls over their own stores, replayed at the same time, give what the calls gave one after the other."""
    torch = require_cuda()
    import vla_cpp_b200 as vb

    B, P, S, n_q, n_kv, hd, keep = 2, 700, 7, 4, 1, 128, 300
    freqs, m = vb.rope_freqs(hd)

    def build(seed):
        x, (wq, wk), lens, g = prompts(torch, B, P, n_q, n_kv, hd, seed)
        st, small = vb.KvStore(1, B, n_kv, hd, 0, P), vb.KvStore(1, B, n_kv, hd, keep, 0)
        xs = torch.randn(B * S, n_q * hd, device="cuda", generator=g).bfloat16()
        row0 = torch.zeros(B, dtype=torch.int32, device="cuda")

        def calls():
            vb.qk_norm_rope_append(st, 0, x, P, n_q, freqs, wq, wk, row0=row0, n_tok=lens)
            q = vb.qk_norm_rope_append(st, 0, xs, S, n_q, freqs, wq, with_kv=False)
            out, lse = vb.cross_attention(st, 0, q, lens=lens)  # few units, many blocks: through the workspace
            mass = vb.key_mass(st, 0, q, lse, lens=lens)
            left, kept, weights = vb.kv_evict(st, small, mass[None], keep, lens=lens, recent=5)
            out2, lse2 = vb.cross_attention(small, 0, q, lens=left)
            return q, out, lse, mass, left, kept, weights, out2, lse2

        return calls, small

    made = [build(s) for s in (1, 2)]
    want = [[t.clone() for t in calls()] + [small.k.clone(), small.v.clone()] for calls, small in made]
    torch.cuda.synchronize()
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in made]
    for calls, _ in made:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(calls())
        graphs.append(graph)
    for _ in range(5):
        for (_, small), res in zip(made, outs):
            small.k.zero_()
            small.v.zero_()
            for t in res:
                t.zero_()
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for (_, small), res, w in zip(made, outs, want):
            for a, b in zip([*res, small.k, small.v], w):
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert vb.device_status() == 0


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_one_token_replayed_while_the_cache_grows(hd):
    """A captured step -- rotate and append at row0, attend over row0 + 1 rows -- replayed as the lengths move on, against the calls."""
    torch = require_cuda()
    import vla_cpp_b200 as vb

    B, n_q, n_kv, cap = 3, 8, 2, 4000
    g = torch.Generator(device="cuda").manual_seed(hd)
    st, other = vb.KvStore(1, B, n_kv, hd, 0, cap), vb.KvStore(1, B, n_kv, hd, 0, cap)
    for t in (st.k, st.v):
        t.normal_(0, 1, generator=g)
    other.k.copy_(st.k)
    other.v.copy_(st.v)
    freqs, m = vb.rope_freqs(hd)
    x = torch.empty(B, (n_q + 2 * n_kv) * hd, dtype=torch.bfloat16, device="cuda")
    row0, lens = (torch.zeros(B, dtype=torch.int32, device="cuda") for _ in range(2))
    mass = torch.zeros(B, n_kv, cap, device="cuda")

    def step(store, weights):
        q = vb.qk_norm_rope_append(store, 0, x, 1, n_q, freqs, row0=row0)
        out, lse = vb.cross_attention(store, 0, q, lens=lens)
        vb.key_mass(store, 0, q, lse, lens=lens, mass=weights, out=weights)
        return out, lse

    x.zero_()
    for store in (st, other):  # the first call is not captured; it writes row 0 of both
        step(store, mass.clone())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(st, mass)
    mine = torch.zeros_like(mass)
    for at in ([0, 0, 63], [1, 64, 64], [127, 128, 700], [3999, 1, 2047], [3999, 3998, 3997]):
        x.normal_(0, 1, generator=g)
        row0.copy_(torch.tensor(at, dtype=torch.int32))
        lens.copy_(row0 + 1)
        if at == [1, 64, 64]:
            lens[0] = 0  # an idle observation
        graph.replay()
        want = step(other, mine)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(mass, mine)
        assert torch.equal(st.k, other.k) and torch.equal(st.v, other.v)
        seen = torch.arange(cap, device="cuda")[None] < lens[:, None]
        q = vb.qk_norm_rope_append(other, 0, x, 1, n_q, freqs, row0=row0)
        z = (q.double().reshape(B, n_kv, -1, hd) @ other.k[0].double().transpose(-1, -2) * hd ** -0.5).masked_fill(~seen[:, None, None], -float("inf"))
        ref = torch.logsumexp(z, -1).reshape(B, n_q, 1)
        assert torch.equal(ref == -float("inf"), got[1] == -float("inf"))
        torch.testing.assert_close(got[1].double().nan_to_num(neginf=0), ref.nan_to_num(neginf=0), rtol=1e-5, atol=1e-5)
    assert vb.device_status() == 0


@pytest.mark.parametrize("hd,S", [(64, 1), (128, 40), (256, 1)])
def test_what_follows_a_call_whose_pieces_are_all_whole(hd, S):
    """max_len asks for cut units, the lengths leave none cut: nothing to merge, and the next call still sees what the first one wrote."""
    torch = require_cuda()
    import vla_cpp_b200 as vb

    B, n_q, n_kv, cap = 20, 6, 2, 6000
    g = torch.Generator(device="cuda").manual_seed(hd)
    st = vb.KvStore(1, B, n_kv, hd, 0, cap)
    st.k.normal_(0, 1, generator=g)
    st.v.normal_(0, 1, generator=g)
    q = torch.randn(B, n_q, S, hd, device="cuda", generator=g).bfloat16()
    lens = torch.full((B,), 128, dtype=torch.int32, device="cuda")
    out, lse = vb.cross_attention(st, 0, q, lens=lens)
    torch.cuda.synchronize()
    want = vb.key_mass(st, 0, q, lse, lens=lens)
    mass = torch.zeros_like(want)
    again = torch.empty_like(lse)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        vb.cross_attention(st, 0, q, lens=lens, out=out, lse=again)
        vb.key_mass(st, 0, q, again, lens=lens, out=mass)
    for _ in range(20):
        again.fill_(3.0)
        mass.zero_()
        graph.replay()
        assert torch.equal(again, lse) and torch.equal(mass, want)
    assert vb.device_status() == 0


def test_denoise_attention_over_an_evicted_cache():
    """The isolated denoise-attention op runs on the smaller store, its action tokens at their old positions."""
    torch = require_cuda()
    import vla_cpp_b200 as vb

    L, B, n_q, n_kv, hd, P, S, H, keep = 2, 3, 15, 5, 64, 177, 51, 320, 77
    g = torch.Generator(device="cuda").manual_seed(5)
    st, small, by_hand = vb.KvStore(L, B, n_kv, hd, P, S), vb.KvStore(L, B, n_kv, hd, keep, S), vb.KvStore(L, B, n_kv, hd, keep, S)
    for l in range(L):
        st.write_prefix(l, *(torch.randn(B, P, n_kv, hd, device="cuda", generator=g) for _ in range(2)))
    mass = torch.rand(L, B, n_kv, st.cap, device="cuda", generator=g)
    _, kept, _ = vb.kv_evict(st, small, mass, keep, max_len=P)
    for l in range(L):
        for b in range(B):
            for h in range(n_kv):
                rows = kept[l, b, h].long()
                by_hand.k[l, b, h, :keep] = st.k[l, b, h, rows]
                by_hand.v[l, b, h, :keep] = st.v[l, b, h, rows]
    ln = torch.ones(L, H, device="cuda")
    w = (torch.randn(L, (n_q + 2 * n_kv) * hd, H, device="cuda", generator=g) * 0.02).bfloat16()
    x = torch.randn(1, L, B * S, H, device="cuda", generator=g).bfloat16()
    a, b = (vb.DenoiseAttn(s, H, n_q, S, ln, w, 1e-5, vb.MASK_CAUSAL, pos0=P).run(x) for s in (small, by_hand))
    assert vb.device_status() == 0
    assert torch.equal(a, b) and torch.equal(small.k, by_hand.k) and torch.equal(small.v, by_hand.v)


def test_large_offsets():
    """Pages beyond 2^32 elements from the start of the store: the last observation's are the ones written, read, weighed and moved."""
    torch = require_cuda()
    import vla_cpp_b200 as vb

    B, n_kv, hd, cap = 33, 1, 128, 1 << 20  # 33 x 2^27 elements of K: 8.9 GB, twice
    S, n_q, keep = 2, 2, 3
    st, small = vb.KvStore(1, B, n_kv, hd, 0, cap), vb.KvStore(1, B, n_kv, hd, keep, 0)
    g = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn(B * S, (n_q + 2 * n_kv) * hd, device="cuda", generator=g).bfloat16()
    row0 = torch.zeros(B, dtype=torch.int32, device="cuda")
    row0[-1] = cap - S
    q = vb.qk_norm_rope_append(st, 0, x, S, n_q, row0=row0)
    assert torch.equal(st.k[0, -1, 0, -S:], x[-S:, n_q * hd:(n_q + 1) * hd]) and torch.equal(st.v[0, -1, 0, -S:], x[-S:, (n_q + 1) * hd:])
    lens = torch.full((B,), S, dtype=torch.int32, device="cuda")
    lens[-1] = cap
    out, lse = vb.cross_attention(st, 0, q, lens=lens)
    # a million rows of zero and the last two: the score of a zero row is 0
    z = (q[-1].double() @ st.k[0, -1, 0, -S:].double().T) * hd ** -0.5
    total = torch.exp(z).sum(-1) + (cap - S)
    torch.testing.assert_close(lse[-1].double(), torch.log(total), rtol=1e-5, atol=0)
    want = (torch.exp(z) / total[..., None]) @ st.v[0, -1, 0, -S:].double()
    err = (out[-1].double().reshape(S, n_q, hd).transpose(0, 1) - want).abs()
    assert bool((err <= 2.0 ** -7 * ((torch.exp(z) / total[..., None]) @ st.v[0, -1, 0, -S:].double().abs())).all())
    mass = vb.key_mass(st, 0, q, lse, lens=lens)
    torch.testing.assert_close(mass[-1, 0, -S:].double(), (torch.exp(z) / total[..., None]).sum((0, 1)), rtol=1e-4, atol=0)
    _, kept, _ = vb.kv_evict(st, small, mass[None], keep, lens=lens, recent=2)
    assert kept[0, -1, 0, 1:].tolist() == [cap - 2, cap - 1]
    assert torch.equal(small.k[0, -1, 0, 1:], st.k[0, -1, 0, -2:]) and vb.device_status() == 0

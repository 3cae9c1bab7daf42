"""A query row whose log-sum-exp is -inf weighs nothing, whatever stands in the row and in the pages: an idle token's query that nobody wrote, or a
score that is infinite."""
import math

import pytest

from tests.gpu_util import require_cuda
from tests.test_key_mass import make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,S,n_q,n_kv,hd,cap,lens", [
    (2, 1, 8, 1, 256, 300, [300, 129]),
    (3, 7, 6, 2, 64, 260, [260, 0, 100]),
    (2, 70, 4, 1, 128, 400, [400, 257]),     # 280 rows: two chunks
    (2, 33, 8, 1, 256, 300, [1, 300]),       # 264 rows: three
    (90, 40, 4, 1, 64, 300, [300] * 90),     # several units per pair
])
def test_rows_that_saw_nothing_weigh_nothing(B, S, n_q, n_kv, hd, cap, lens):
    torch = require_cuda()
    import vla_cpp_b200 as vb

    st, q, lens, _, g = make(torch, B, S, n_q, n_kv, hd, cap, lens, False, 5, layers=1)
    lse = torch.randn(B, n_q, S, device="cuda", generator=g) + 6.0
    idle = torch.rand(B, n_q, S, device="cuda", generator=g) < 0.4
    idle[0, 0, 0], idle[-1, -1, -1] = True, True
    lse[idle] = -math.inf
    mass = torch.rand(B, n_kv, cap, device="cuda", generator=g)
    q[idle] = 0.0
    want = vb.key_mass(st, 0, q, lse, lens=lens, mass=mass)
    for junk in (math.nan, math.inf, -math.inf, 3e38):
        q[idle] = junk
        got = vb.key_mass(st, 0, q, lse, lens=lens, mass=mass)
        assert torch.equal(got, want), junk
    # an infinite element of a cached row: rows that did see something have their NaN or infinity, those that did not none
    lse.fill_(-math.inf)
    q.normal_(0, 1, generator=g)
    st.k[..., 0] = math.inf
    st.k[..., 1] = math.nan
    live = (torch.arange(cap, device="cuda")[None] < lens[:, None])[:, None].expand_as(mass)
    assert torch.equal(vb.key_mass(st, 0, q, lse, lens=lens, mass=mass), torch.where(live, mass, 0.0))
    assert vb.device_status() == 0

"""Arguments of the ragged cache calls that are no tensors, or ask for more rows than there are, are refused as the other wrong ones are: by VlaB200Error,
before anything is allocated for them."""
import pytest

from tests.gpu_util import require_cuda

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("freqs", [[1.0, 0.5], 3, "no", (None,)])
def test_angles_that_are_no_tensor(freqs):
    torch = require_cuda()
    import vla_cpp_b200 as vb

    st = vb.KvStore(1, 1, 1, 64, 4, 0)
    x = torch.zeros(2, 3 * 64, device="cuda")
    with pytest.raises(vb.VlaB200Error) as e:
        vb.qk_norm_rope_append(st, 0, x, 2, 1, freqs)
    assert e.value.code == -1


def test_angles_of_two_dimensions():
    torch = require_cuda()
    import vla_cpp_b200 as vb

    st = vb.KvStore(1, 1, 1, 64, 4, 0)
    x = torch.zeros(2, 3 * 64, device="cuda")
    with pytest.raises(vb.VlaB200Error):
        vb.qk_norm_rope_append(st, 0, x, 2, 1, torch.zeros(2, 4, dtype=torch.float64, device="cuda"))


def test_more_rows_kept_than_the_smaller_store_has():
    torch = require_cuda()
    import vla_cpp_b200 as vb

    src, dst = vb.KvStore(1, 1, 1, 64, 50, 0), vb.KvStore(1, 1, 1, 64, 20, 0)
    mass = torch.zeros(1, 1, 1, 50, device="cuda")
    for keep in (21, 2 ** 31 - 1, 2 ** 40):
        with pytest.raises(vb.VlaB200Error) as e:
            vb.kv_evict(src, dst, mass, keep)
        assert e.value.code == -1
